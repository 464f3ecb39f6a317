"""Token operators on the GPU against their formulas in float64 (oracle/attention.py), within bounds that follow from the roundings."""
import math
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "droid-slam_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

from droid_amd import attention as at  # noqa: E402
from oracle import attention as oa  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def near(got, want, err, what):
    got, want = got.detach().double().cpu(), want.detach()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(nan=7e300, posinf=5e300, neginf=-5e300), want[~fine].nan_to_num(nan=7e300, posinf=5e300, neginf=-5e300)), what
    over = ((got - want).abs() - err)[fine]
    assert over.numel() == 0 or over.max() <= 0, "%s: off by up to %.3g where %.3g is allowed" % (what, (got - want).abs()[fine].max(), err[fine].max())


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def inputs(lengths, key_lengths, heads, kv_heads, dim, dtype, seed=0, pad=0):
    m, l = sum(lengths) + pad, sum(key_lengths if key_lengths is not None else lengths) + pad
    return (rand((m, heads, dim), dtype, seed, 1.5), rand((l, kv_heads, dim), dtype, seed + 1), rand((l, kv_heads, dim), dtype, seed + 2) + 0.25, rand((m, heads, dim), dtype, seed + 3))


#        lengths, key lengths, heads, kv_heads, dim, block
CASES = [([1], None, 1, 1, 8, 0), ([1], None, 4, 4, 32, 1), ([2, 1, 0, 3], None, 2, 2, 64, 1), ([48], None, 4, 4, 32, 0), ([33, 64, 65], None, 4, 2, 64, 1),
         ([127, 129], None, 2, 2, 128, 1), ([200], None, 8, 2, 128, 0), ([96], None, 6, 2, 40, 16), ([150, 31], None, 32, 1, 16, 7), ([70], None, 3, 1, 80, 1),
         ([257], None, 5, 5, 24, 100), ([60, 5, 0, 20], [20, 50, 9, 0], 4, 4, 64, 1), ([60], [20], 4, 2, 96, 8), ([5, 40], [300, 41], 4, 2, 128, 1),
         ([192 * 3], None, 4, 2, 64, 192), ([3, 9, 1], [200, 77, 640], 2, 1, 104, 0), ([500], [130], 2, 2, 64, 0)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,key_lengths,heads,kv_heads,dim,block", CASES)
def test_attention_and_gradients(lengths, key_lengths, heads, kv_heads, dim, block, dtype):
    q, k, v, g = inputs(lengths, key_lengths, heads, kv_heads, dim, dtype)
    plan = at.PackedPlan(lengths, heads, kv_heads, dim, key_lengths=key_lengths, causal_block=block)
    r = oa.attention(q, k, v, lengths, key_lengths, block=block, grad=g)
    o, lse = at.packed_attention(q, k, v, plan, return_lse=True)
    near(o, r["o"], r["o_err"], "o")
    near(lse, r["lse"], r["lse_err"], "lse")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = at.packed_attention(*leaves, plan)
    assert torch.equal(out, o)
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 16, 2, 128), (F16, 4, 4, 64), (BF16, 3, 3, 40), (F16, 32, 1, 128), (F16, 6, 1, 32)])
@pytest.mark.parametrize("block", [0, 1, 50])
def test_few_queries_over_long_keys(dtype, heads, kv_heads, dim, block):
    """rows that are split over their keys and joined; single queries, some with one key or none"""
    lengths, keys = [1, 1, 2, 1, 1, 1], [1, 5000, 2047, 0, 64, 12345]
    q, k, v, g = inputs(lengths, keys, heads, kv_heads, dim, dtype, 5)
    plan = at.PackedPlan(lengths, heads, kv_heads, dim, key_lengths=keys, causal_block=block)
    assert int(plan.info[7]) > 0 and int(plan.info[9]) > 0                   # (rows split in the forward and in the backward)
    r = oa.attention(q, k, v, lengths, keys, block=block, grad=g)
    o, lse = at.packed_attention(q, k, v, plan, return_lse=True)
    near(o, r["o"], r["o_err"], "o")
    near(lse, r["lse"], r["lse_err"], "lse")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(at.packed_attention(*leaves, plan), leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_views_and_padding(dtype):
    """heads sliced from one projection, heads outside tokens, broadcast key heads, unaligned views, rows behind the last sequence"""
    lengths, heads, kv, d = [70, 30], 4, 2, 64
    qkv = rand((120, heads + 2 * kv, d), dtype, 1)
    qkv[100:] = float("nan")                                                 # behind the last sequence: never read
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    g = rand((120, heads, d), dtype, 2)
    plan = at.PackedPlan(lengths, heads, kv, d, causal_block=1)
    r = oa.attention(q[:100], k[:100], v[:100], lengths, block=1, grad=g[:100])

    def check(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = at.packed_attention(*leaves, plan)
        near(o[:100], r["o"], r["o_err"], "o")
        assert not o[100:].any()
        for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
            near(t[:100], r[n], r[n + "_err"], n)
            assert t.shape[0] == 120 and not t[100:].any()

    check(q, k, v, g)
    check(*[t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)])       # [heads, tokens, d] in memory
    odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731  (an address that is no multiple of 16)
    check(odd(q), odd(k), odd(v), odd(g))
    check(*[torch.stack([t, t], -1)[..., 0] for t in (q, k, v, g)])          # channels not adjacent
    same = k[:1].expand(120, -1, -1)                                         # one row of keys seen by all tokens: its gradient is a sum
    r0 = oa.attention(q[:100], same[:100], v[:100], lengths, block=1, grad=g[:100])
    leaf = k[:1].detach().clone().requires_grad_()
    (dk,) = torch.autograd.grad(at.packed_attention(q, leaf.expand(120, -1, -1), v, plan), leaf, g)
    near(dk, r0["dk"].sum(0, keepdim=True), r0["dk_err"].sum(0, keepdim=True) + 100 * oa.half_step(dtype) * r0["dk"].abs().sum(0, keepdim=True), "dk of a broadcast row")
    one = k[:, :1].expand(-1, kv, -1)                                        # one key head read by all: its gradient is a sum
    r1 = oa.attention(q[:100], one[:100], v[:100], lengths, block=1, grad=g[:100])
    leaf = k[:, :1].detach().clone().requires_grad_()
    o = at.packed_attention(q, leaf.expand(-1, kv, -1), v, plan)
    (dk,) = torch.autograd.grad(o, leaf, g)
    u = oa.half_step(dtype)
    near(dk[:100], r1["dk"].sum(1, keepdim=True), r1["dk_err"].sum(1, keepdim=True) + 2 * u * r1["dk"].abs().sum(1, keepdim=True), "dk of a broadcast head")
    grad = torch.autograd.grad(at.packed_attention(leaf.expand(-1, heads, -1), k, v, plan).float().sum(), leaf)[0]    # a gradient without strides
    assert torch.isfinite(grad[:100]).all()


def test_out_is_written_only_where_sequences_are():
    q, k, v, _ = inputs([40, 7], None, 4, 4, 64, F16, pad=5)
    plan = at.PackedPlan([40, 7], 4, 4, 64, causal_block=1)
    want = at.packed_attention(q, k, v, plan)
    buf = torch.full((52, 6, 64), 3.0, dtype=F16, device="cuda")
    got = at.packed_attention(q, k, v, plan, out=buf[:, 1:5])
    assert got.data_ptr() == buf[:, 1:5].data_ptr() and torch.equal(got[:47], want[:47])
    assert bool((buf[47:] == 3).all()) and bool((buf[:, 0] == 3).all()) and bool((buf[:, 5] == 3).all())
    for bad in (q, buf[:, 0:4, :32], buf[:, 1:5].float(), buf[:51, 1:5], k, torch.empty(1, 4, 64, dtype=F16, device="cuda").expand(52, -1, -1)):
        with pytest.raises(RuntimeError):
            at.packed_attention(q, k, v, plan, out=bad)
    with pytest.raises(RuntimeError, match="gradient"):
        at.packed_attention(q.requires_grad_(), k, v, plan, out=buf[:, 1:5])


def test_keys_in_slots_of_a_cache():
    """key_starts: sequences read their slots; shared keys are allowed forward and refused backward; unused rows get zero gradients"""
    heads, kv, d, cap = 4, 2, 64, 200
    q, _, _, g = inputs([1, 3, 20], None, heads, kv, d, BF16)
    k, v = rand((3 * cap, kv, d), BF16, 11), rand((3 * cap, kv, d), BF16, 12)
    keys, starts = [130, 3, 77], [2 * cap, 0, cap]
    used = torch.zeros(3 * cap, dtype=torch.bool)
    for a, n in zip(starts, keys):
        used[a:a + n] = True
    k[~used.cuda()], v[~used.cuda()] = float("inf"), float("nan")
    plan = at.PackedPlan([1, 3, 20], heads, kv, d, key_lengths=keys, key_starts=starts, causal_block=1)
    r = oa.attention(q, k, v, [1, 3, 20], keys, starts, block=1, grad=g)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = at.packed_attention(*leaves, plan)
    near(o, r["o"], r["o_err"], "o")
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
        near(t, r[n], r[n + "_err"], n)
        if n != "dq":
            assert not t.cpu()[~used].any()
    starts = [0, 0, 10]
    k, v = rand((cap, kv, d), BF16, 13), rand((cap, kv, d), BF16, 14)
    plan = at.PackedPlan([1, 3, 20], heads, kv, d, key_lengths=keys, key_starts=starts)
    r = oa.attention(q, k, v, [1, 3, 20], keys, starts)
    near(at.packed_attention(q, k, v, plan), r["o"], r["o_err"], "o of shared keys")
    with pytest.raises(RuntimeError, match="share"):
        torch.autograd.grad(at.packed_attention(q.requires_grad_(), k, v, plan), q, g)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,n", [(64, 150), (128, 70), (32, 300)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, d, n):
    q, k, v, _ = inputs([n], None, 2, 1, d, dtype, 3)
    plan = at.PackedPlan([n], 2, 1, d, causal_block=1)
    clean = at.packed_attention(q, k, v, plan)
    at_inf, at_nan = n // 2, n - 20
    bad = v.clone()
    bad[at_inf, 0, 3], bad[at_inf, 0, 5], bad[at_nan, 0, 7], bad[at_nan, 0, 3] = float("inf"), -float("inf"), float("nan"), -float("inf")
    o = at.packed_attention(q, k, bad, plan)
    assert torch.equal(o[:at_inf], clean[:at_inf])
    assert bool((o[at_inf:at_nan, :, 3] == float("inf")).all()) and bool((o[at_inf:, :, 5] == -float("inf")).all())
    assert bool(o[at_nan:, :, 7].isnan().all()) and bool(o[at_nan:, :, 3].isnan().all())
    others = [c for c in range(d) if c not in (3, 5, 7)]
    assert torch.equal(o[:, :, others], clean[:, :, others])
    bad = k.clone()
    bad[at_nan, 0, 1], bad[at_inf, 0, 0] = float("nan"), -float("inf")       # a key: rows before it do not change
    o = at.packed_attention(q, bad, v, plan)
    assert torch.equal(o[:at_inf], clean[:at_inf]) and bool(o[at_nan:].isnan().all())
    bad = q.clone()
    bad[at_inf, 1] = float("nan")                                            # a query: its own row only
    o = at.packed_attention(bad, k, v, plan)
    assert bool(o[at_inf, 1].isnan().all()) and torch.equal(o[:at_inf], clean[:at_inf]) and torch.equal(o[at_inf + 1:], clean[at_inf + 1:])


@pytest.mark.parametrize("scale", [None, 1.0, 0.01])
def test_large_scores_and_scale(scale):
    """scores far apart and far from zero: a running maximum has to carry them"""
    q, k, v, g = inputs([200], None, 2, 2, 64, BF16, 9)
    q, k = q * 4, k * 4
    k[100:] *= 3                                                             # the maximum grows late
    plan = at.PackedPlan([200], 2, 2, 64)
    r = oa.attention(q, k, v, [200], scale=scale, grad=g)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = at.packed_attention(*leaves, plan, scale=scale)
    near(o, r["o"], r["o_err"], "o")
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,lengths,keys,block", [(BF16, 8, 1, 128, [6000, 40], [30, 200], 0), (F16, 16, 1, 64, [700], [640], 320),
                                                                         (BF16, 3, 1, 32, [9000], [9], 0), (F16, 2, 1, 104, [8000], [260], 0)])
def test_many_rows_over_few_keys(dtype, heads, kv_heads, dim, lengths, keys, block):
    """gradients of keys that are split over their rows and joined"""
    q, k, v, g = inputs(lengths, keys, heads, kv_heads, dim, dtype, 6)
    plan = at.PackedPlan(lengths, heads, kv_heads, dim, key_lengths=keys, causal_block=block)
    assert int(plan.info[11]) > 0                                            # (split keys)
    r = oa.attention(q, k, v, lengths, keys, block=block, grad=g)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = at.packed_attention(*leaves, plan)
    near(o, r["o"], r["o_err"], "o")
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_as_large_as_they_may_be(sign, dtype):
    """scores of 2.5 10^7 and 5 10^7, of either sign, far apart: one key's weight is one"""
    q = torch.full((3, 2, 64), 2048.0, dtype=dtype, device="cuda")
    k = torch.full((3, 1, 64), sign * 1536.0, dtype=dtype, device="cuda")
    k[1] *= 2 if sign > 0 else 0.5                                           # the second key wins wherever it is seen
    v = rand((3, 1, 64), dtype, 1)
    o, lse = at.packed_attention(q, k, v, at.PackedPlan([3], 2, 1, 64, causal_block=1), return_lse=True)
    for i, winner in enumerate((0, 1, 1)):
        assert torch.equal(o[i], v[winner].expand(2, -1)), i
    assert bool(torch.isfinite(lse).all())


def test_attention_gradient_against_differences():
    """the kernels' gradients against central differences of the float64 forward along random directions"""
    lengths, heads, kv, d = [40, 9], 4, 2, 32
    q, k, v, g = inputs(lengths, None, heads, kv, d, F16, 21)
    plan = at.PackedPlan(lengths, heads, kv, d, causal_block=4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(at.packed_attention(*leaves, plan), leaves, g)
    r = oa.attention(q, k, v, lengths, block=4, grad=g)
    for n, name in enumerate(("dq", "dk", "dv")):
        x = torch.randn(leaves[n].shape, generator=torch.Generator().manual_seed(n), dtype=torch.float64)
        t = [a.double().cpu() for a in (q, k, v)]
        f = []
        for h in (1e-4, -1e-4):
            t2 = list(t)
            t2[n] = t[n] + h * x
            f.append((oa.attention(*t2, lengths, block=4)["o"] * g.double().cpu()).sum())
        want = (f[0] - f[1]) / 2e-4
        allowed = (r[name + "_err"] * x.abs()).sum() + 1e-5
        assert abs((grads[n].double().cpu() * x).sum() - want) <= allowed, name


def test_same_bits_every_time_and_on_streams():
    """no result depends on timing: repeated, on side streams at once, and captured and replayed with other work between"""
    lengths, keys, heads, kv, d = [300, 1, 77], [300, 9000, 500], 8, 2, 64
    sets = [inputs(lengths, keys, heads, kv, d, BF16, 30 + 10 * i) for i in range(2)]
    plan = at.PackedPlan(lengths, heads, kv, d, key_lengths=keys, causal_block=1)

    def step(q, k, v, g):
        o, lse, low = at.droid_backends.attention_forward(q, k, v, plan.items, plan.info, 0.125, None, True)
        return (o, lse) + tuple(at.droid_backends.attention_backward(g, q, k, v, o, lse, low, plan.items, plan.info, 0.125))

    want = [step(*s) for s in sets]
    for i in range(3):
        for s, w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(step(*s), w))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([step(*s) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, runs in zip(want, got) for run in runs for a, b in zip(run, w))
    graphs = []
    for s in sets:
        static = [t.clone() for t in s]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(*static)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for i in range(4):
        for n, (graph, static, out) in enumerate(graphs):
            for t, new in zip(static, sets[(n + i) % 2]):
                t.copy_(new)
            graph.replay()
            step(*sets[0])                                                   # eager work between the replays
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[(n + i) % 2])), (n, i)


def test_captured_training_step():
    """forward and autograd's backward in one graph, replayed on new inputs"""
    lengths, heads, kv, d = [96, 33], 4, 2, 64
    plan = at.PackedPlan(lengths, heads, kv, d, causal_block=1)
    pos, fr, w = torch.arange(129, device="cuda", dtype=torch.int32), torch.rand(32, device="cuda"), torch.rand(d, device="cuda")

    def step(q, k, v, g, w):
        a, b = at.qk_norm_rope(q, k, pos, fr, [32], w, w)
        return torch.autograd.grad(at.packed_attention(a, b, v, plan), (q, k, v, w), g)

    sets = [inputs(lengths, None, heads, kv, d, BF16, 40 + 10 * i) for i in range(2)]
    leaf = lambda s: [t.clone().requires_grad_() for t in s[:3]] + [s[3].clone(), w.clone().requires_grad_()]  # noqa: E731
    want = [step(*leaf(s)) for s in sets]
    static = leaf(sets[0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(*static)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for i in range(4):
        with torch.no_grad():
            for t, new in zip(static, sets[i % 2]):
                t.copy_(new)
        graph.replay()
        step(*leaf(sets[0]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2])), i


def test_capture_beside_a_living_graph_of_the_same_leaves_is_refused():
    q, k, v, g = inputs([40], None, 4, 2, 64, BF16)
    plan = at.PackedPlan([40], 4, 2, 64, causal_block=1)
    pos, fr = torch.arange(40, device="cuda", dtype=torch.int32), torch.rand(32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    alive = at.packed_attention(*leaves, plan)
    for call in (lambda: at.packed_attention(*leaves, plan), lambda: at.qk_norm_rope(leaves[0], leaves[1], pos, fr, [32])):
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    want = torch.autograd.grad(alive, leaves, g)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(at.packed_attention(*leaves, plan), leaves, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_beyond_32_bits():
    """rows that lie more than 4 GiB from the start: far slots of a cache, and token strides of 16 MB"""
    h, kv, d, far = 4, 2, 64, 20000000
    cache = [torch.empty(far + 300, kv, d, dtype=BF16, device="cuda") for _ in range(2)]
    assert far * kv * d * 2 > 1 << 32
    q, k, v, g = inputs([5, 200], [5, 300], h, kv, d, BF16, 50)
    for c, t in zip(cache, (k, v)):
        c[:5], c[far:] = t[:5], t[5:]
    plan = at.PackedPlan([5, 200], h, kv, d, key_lengths=[5, 300], key_starts=[0, far], causal_block=1)
    r = oa.attention(q, k, v, [5, 200], [5, 300], block=1, grad=g)
    leaves = [q.clone().requires_grad_()] + [c.requires_grad_() for c in cache]
    o = at.packed_attention(*leaves, plan)
    near(o, r["o"], r["o_err"], "o")
    grads = torch.autograd.grad(o, leaves, g)
    near(grads[0], r["dq"], r["dq_err"], "dq")
    for n, t in zip(("dk", "dv"), grads[1:]):
        near(torch.cat([t[:5], t[far:]]), r[n], r[n + "_err"], n)
        assert not t[5:200].any()
    del cache, leaves, grads
    n, st = 330, 8000000                                                     # elements between tokens
    assert n * st * 2 > 1 << 32
    wide = torch.empty(n * st, dtype=BF16, device="cuda")
    lay = lambda t, at_: wide.as_strided(t.shape, (st, t.shape[2], 1), at_).copy_(t)  # noqa: E731
    q, k, v, g = inputs([n], None, h, kv, d, BF16, 60)
    r = oa.attention(q, k, v, [n], block=1, grad=g)
    Q, K, V, G = lay(q, 0), lay(k, 1024), lay(v, 2048), lay(g, 4096)
    plan = at.PackedPlan([n], h, kv, d, causal_block=1)
    out = wide.as_strided(q.shape, (st, d, 1), 8192)
    near(at.packed_attention(Q, K, V, plan, out=out), r["o"], r["o_err"], "o")
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(at.packed_attention(*leaves, plan), leaves, G)):
        near(t, r[name], r[name + "_err"], name)
    pos, fr = torch.arange(n).int().cuda(), torch.rand(32).cuda()
    rq = oa.qk_norm_rope(q, pos, fr, [32], grad=g)
    y = at.qk_norm_rope(Q, K, pos, fr, [32], out=(out, wide.as_strided(k.shape, (st, d, 1), 16384)))
    near(y[0], rq["y"], rq["y_err"], "rotation")


def test_nothing_on_one_side():
    """keys without queries get zero gradients, queries without keys zero results and gradients; the same tensor may be all three inputs"""
    q, k, v, g = inputs([0, 6], [5, 0], 4, 2, 64, BF16)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = at.packed_attention(*leaves, at.PackedPlan([0, 6], 4, 2, 64, key_lengths=[5, 0], causal_block=1), return_lse=True)
    assert not o.any() and bool((lse == -math.inf).all()) and not lse.requires_grad
    assert all(not t.any() for t in torch.autograd.grad(o, leaves, g))
    k, v = rand((300, 2, 64), BF16, 1).requires_grad_(), rand((300, 2, 64), BF16, 2).requires_grad_()
    q = rand((4, 4, 64), BF16, 3).requires_grad_()                           # no sequence at all has queries
    o = at.packed_attention(q, k, v, at.PackedPlan([0], 4, 2, 64, key_lengths=[300]))
    assert not o.any() and all(not t.any() for t in torch.autograd.grad(o, (q, k, v), g[:4]))
    x = rand((50, 3, 64), F16, 4).requires_grad_()
    g = rand((50, 3, 64), F16, 5)
    r = oa.attention(x.detach(), x.detach(), x.detach(), [50], block=1, grad=g)
    (dx,) = torch.autograd.grad(at.packed_attention(x, x, x, at.PackedPlan([50], 3, 3, 64, causal_block=1)), x, g)
    u = oa.half_step(F16)
    near(dx, r["dq"] + r["dk"] + r["dv"], sum(r[n + "_err"] + 2 * u * r[n].abs() for n in ("dq", "dk", "dv")), "dx")
    a, b = at.qk_norm_rope(x, x[:, :0], torch.arange(50, device="cuda"), torch.ones(32, device="cuda"), [32])
    assert a.shape == x.shape and b.shape == (50, 0, 64)
    torch.autograd.grad(a.float().square().sum(), x)


@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_see_nothing_may_hold_anything(d):
    """NaN queries and gradients in rows whose mask leaves nothing: results and gradients are those of finite rows"""
    q, k, v, g = inputs([300], [170], 4, 2, d, BF16, 80)
    plan = at.PackedPlan([300], 4, 2, d, key_lengths=[170], causal_block=1)

    def step(q, g):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = at.packed_attention(*leaves, plan)
        return [o] + list(torch.autograd.grad(o, leaves, g))

    want = step(q, g)
    q[:130], g[:130] = float("nan"), float("nan")
    got = step(q, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][:130].any() and not got[1][:130].any()


def test_raw_c_abi_on_a_side_stream():
    """the C entries with plain pointers on a stream of the caller's: the binding's bits, rows behind the sequences left as they were"""
    import ctypes
    from tests.test_attention_cpu import FIELDS
    lib = ctypes.CDLL(os.path.join(os.path.dirname(at.droid_backends.__file__), "libdroid_hip.so"))
    i64, ptr, f32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    for name in ("dh_attn_fwd_workspace_bytes", "dh_attn_bwd_workspace_bytes", "dh_qk_norm_rope_bwd_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    lengths, keys, h, kv, d, pad = [1, 4, 2], [9000, 30, 5000], 4, 2, 64, 3
    q, k, v, g = inputs(lengths, keys, h, kv, d, F16, 70, pad)
    plan = at.PackedPlan(lengths, h, kv, d, key_lengths=keys, causal_block=1)
    o, lse, low = at.droid_backends.attention_forward(q, k, v, plan.items, plan.info, 0.125, None, True)
    want = [o, lse] + at.droid_backends.attention_backward(g, q, k, v, o, lse, low, plan.items, plan.info, 0.125)
    info = (i64 * len(FIELDS))()
    ql, kl = (i64 * 3)(*lengths), (i64 * 3)(*keys)
    assert lib.dh_attn_plan(ql, kl, None, i64(3), h, kv, d, i64(1), None, i64(0), info) == 0
    items = (ctypes.c_int32 * info[0])()
    assert lib.dh_attn_plan(ql, kl, None, i64(3), h, kv, d, i64(1), items, i64(info[0]), info) == 0
    items = torch.frombuffer(items, dtype=torch.int32).clone().cuda()
    o2, lse2, dq, dk, dv = [torch.full_like(t, 7.0) for t in want]
    low2 = torch.empty_like(o2)
    wf, wb = lib.dh_attn_fwd_workspace_bytes(info), lib.dh_attn_bwd_workspace_bytes(info)
    ws = torch.empty(max(wf, wb) + 16, dtype=torch.uint8, device="cuda")
    t = lambda x: (ptr(x.data_ptr()), i64(x.stride(0)), i64(x.stride(1)))  # noqa: E731
    p = lambda x: ptr(x.data_ptr())  # noqa: E731
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    tail = (p(items), info, 0, i64(q.shape[0]), i64(k.shape[0]), f32(0.125), 0, p(ws))
    assert lib.dh_attn_fwd(*t(q), *t(k), *t(v), *t(o2), p(low2), p(lse2), *tail, ctypes.c_size_t(wf), ptr(st.cuda_stream)) == 0
    assert lib.dh_attn_bwd(*t(g), *t(q), *t(k), *t(v), *t(o2), p(low2), p(lse2), *t(dq), *t(dk), *t(dv), *tail, ctypes.c_size_t(wb), ptr(st.cuda_stream)) == 0
    st.synchronize()
    for a, b, n in zip((o2, lse2, dq, dk, dv), want, (sum(lengths),) * 3 + (sum(keys),) * 2):
        assert torch.equal(a[:n], b[:n]) and bool((a[n:] == 7).all())
    pos, fr, w, sec = torch.arange(len(q)).int().cuda(), torch.rand(32).cuda(), torch.rand(d).cuda(), (ctypes.c_int * 4)(32, 0, 0, 0)
    kk = k[:len(q)]
    want = list(at.qk_norm_rope(q, kk, pos, fr, [32], w, w)) + at.droid_backends.qk_norm_rope_backward(g, kk, q, kk, pos, fr, [32], w, w, True, 1e-6, False)
    got = [torch.empty_like(x) for x in want]
    tail = (p(pos), 0, p(fr), sec, 1, p(w), p(w), 1, 0, i64(len(q)), h, kv, d, 1, f32(1e-6), 0)
    torch.cuda.synchronize()
    assert lib.dh_qk_norm_rope_fwd(*t(q), *t(kk), *t(got[0]), *t(got[1]), *tail, ptr(st.cuda_stream)) == 0
    n = lib.dh_qk_norm_rope_bwd_workspace_bytes(d)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.dh_qk_norm_rope_bwd(*t(g), *t(kk), *t(q), *t(kk), *t(got[2]), *t(got[3]), p(got[4]), p(got[5]), *tail, p(ws), ctypes.c_size_t(n), ptr(st.cuda_stream)) == 0
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_refusals():
    plan = at.PackedPlan([8], 4, 2, 64)
    q, k, v, g = inputs([8], None, 4, 2, 64, F16)
    for a in ((q.float(), k.float(), v.float()), (q, k.bfloat16(), v), (q[:7], k, v), (q, k[:7], v[:7]), (q, k, v[:, :1]), (q[:, :2], k, v), (q[..., :32], k, v), (q[0], k, v),
              (q, k.cpu(), v), (k, q, q)):
        with pytest.raises(RuntimeError):
            at.packed_attention(*a, plan)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError):
            at.packed_attention(q, k, v, plan, scale=scale)
    with pytest.raises(RuntimeError):
        at.packed_attention(q, k, v, at.PackedPlan([8], 4, 2, 64, device="cpu"))
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(at.packed_attention(leaf, k, v, plan), leaf, g, create_graph=True)
    other = at.PackedPlan([8, 3], 4, 2, 64)
    for info, items in ((other.info, plan.items), (plan.info, other.items), (plan.info[:-1], plan.items), (plan.info.cuda(), plan.items), (torch.zeros_like(plan.info), plan.items)):
        with pytest.raises(RuntimeError):
            at.droid_backends.attention_forward(q, k, v, items, info, 0.1)
    empty = at.PackedPlan([], 4, 2, 64)
    assert not at.packed_attention(q, k, v, empty).any()
    assert at.packed_attention(q[:0], k[:0], v[:0], empty).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------------- norm and rotation
#       tokens, heads, kv_heads, dim, sections
ROPE = [(1, 1, 1, 8, [4]), (48, 4, 4, 32, [4, 6, 6]), (77, 6, 3, 40, [4, 8, 8]), (33, 16, 4, 128, [16, 24, 24]), (50, 3, 1, 64, [5, 0, 7]), (7, 2, 2, 96, [10, 10, 10, 2]),
        (20, 5, 2, 6, [1, 1]), (9, 2, 1, 256, [64, 64]), (130, 1, 8, 80, [20, 20]), (3, 4, 4, 2, [1]), (300, 2, 2, 64, [0])]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("normalize,interleaved", [(True, False), (True, True), (False, False), (False, True)])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,sections", ROPE)
def test_rope_and_gradients(tokens, heads, kv_heads, dim, sections, normalize, interleaved, dtype):
    q, k = rand((tokens, heads, dim), dtype, 1, 2.0), rand((tokens, kv_heads, dim), dtype, 2, 0.5)
    gq, gk = rand((tokens, heads, dim), dtype, 3), rand((tokens, kv_heads, dim), dtype, 4)
    pos = torch.randint(-2000, 100000, (tokens, len(sections)), generator=torch.Generator().manual_seed(5)).int().cuda()
    fr = torch.cat([10000.0 ** (-torch.arange(n) / max(1, n)) for n in sections]).float().cuda()
    wq, wk = (rand((dim,), F32, 6), rand((dim,), F32, 7)) if normalize else (None, None)
    a = dict(positions=pos, inv_freq=fr, sections=sections, normalize=normalize, interleaved=interleaved)
    rq = oa.qk_norm_rope(q, weight=wq, grad=gq, **a)
    rk = oa.qk_norm_rope(k, weight=wk, grad=gk, **a)
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    qo, ko = at.qk_norm_rope(leaves[0], leaves[1], pos, fr, sections, *(leaves[2:] if normalize else (None, None)), normalize=normalize, interleaved=interleaved)
    near(qo, rq["y"], rq["y_err"], "q")
    near(ko, rk["y"], rk["y_err"], "k")
    grads = torch.autograd.grad((qo, ko), leaves, (gq, gk))
    near(grads[0], rq["dx"], rq["dx_err"], "dq")
    near(grads[1], rk["dx"], rk["dx_err"], "dk")
    if normalize:
        near(grads[2], rq["dw"], rq["dw_err"], "dq_weight")
        near(grads[3], rk["dw"], rk["dw_err"], "dk_weight")


@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (F16, F16), (F16, F32), (F32, F32)])
def test_rope_positions_weights_and_views(dtype, wtype):
    n, h, hk, d, sections = 200, 4, 2, 64, [8, 12, 12]
    qkv = rand((n, h + 2 * hk, d), dtype, 1)
    q, k = qkv[:, :h], qkv[:, h:h + hk]
    fr = torch.rand(32).cuda()
    w = rand((d,), wtype, 3)
    far = torch.stack([torch.arange(n) + 1000000, torch.arange(n) * 5, -torch.arange(n)], 1)
    g = [rand(q.shape, dtype, 8), rand(k.shape, dtype, 9)]
    for pos in (far.int().cuda(), far.cuda(), (far.float() + 0.5).cuda()):
        rq = oa.qk_norm_rope(q, pos, fr, sections, weight=w, grad=g[0])
        rk = oa.qk_norm_rope(k, pos, fr, sections, grad=g[1])
        leaves = [q.detach().requires_grad_(), k.detach().requires_grad_(), w.clone().requires_grad_()]
        qo, ko = at.qk_norm_rope(leaves[0], leaves[1], pos, fr, sections, leaves[2])
        near(qo, rq["y"], rq["y_err"], "q")
        near(ko, rk["y"], rk["y_err"], "k")
        for t, want, err in zip(torch.autograd.grad((qo, ko), leaves, g), (rq["dx"], rk["dx"], rq["dw"]), (rq["dx_err"], rk["dx_err"], rq["dw_err"])):
            near(t, want, err, "gradient")
        (alone,) = torch.autograd.grad(at.qk_norm_rope(leaves[0], leaves[1], pos, fr, sections, leaves[2])[0], leaves[0], g[0])      # one result used
        near(alone, rq["dx"], rq["dx_err"], "gradient of q alone")
    pos = far.int().cuda()
    want = at.qk_norm_rope(q, k, pos, fr, sections, w, w)
    rows = torch.zeros(n, 10, d, dtype=dtype, device="cuda")                 # a cache's rows
    with torch.no_grad():
        at.qk_norm_rope(q, k, pos, fr, sections, w, w, out=(rows[:, 1:5], rows[:, 7:9]))
    assert torch.equal(rows[:, 1:5], want[0]) and torch.equal(rows[:, 7:9], want[1]) and not rows[:, [0, 5, 6, 9]].any()
    odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    for a, b in ((odd(q), odd(k)), (q.transpose(0, 1).contiguous().transpose(0, 1), k), (torch.stack([q, q], -1)[..., 0], k)):
        got = at.qk_norm_rope(a, b, pos, fr, sections, w, w)                 # (other lanes hold other channels: sums in another order)
        for t, r in zip(got, [oa.qk_norm_rope(x, pos, fr, sections, weight=w) for x in (q, k)]):
            near(t, r["y"], r["y_err"], "views")
    at.qk_norm_rope(q, k, pos, fr, sections, w, w, out=(q, k))               # in place
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rope_many_tokens_and_repeatable_sums():
    """more tokens than the backward's workgroups hold at once; the weights' gradients are the same bits every time, on any stream, in graphs"""
    n, h, hk, d = 40000, 3, 1, 64
    q, k, gq, gk = rand((n, h, d), BF16, 1), rand((n, hk, d), BF16, 2), rand((n, h, d), BF16, 3), rand((n, hk, d), BF16, 4)
    pos = torch.arange(n).int().cuda()
    fr, w = torch.rand(32).cuda(), rand((d,), F32, 5)
    db = at.droid_backends
    step = lambda: db.qk_norm_rope_backward(gq, gk, q, k, pos, fr, [32], w, w, True, 1e-6, False)  # noqa: E731
    first = step()
    r = oa.qk_norm_rope(q, pos, fr, [32], weight=w, grad=gq)
    near(first[0], r["dx"], r["dx_err"], "dq")
    near(first[2], r["dw"], r["dw_err"], "dw")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        second = step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for i in range(3):
        graph.replay()
        fourth = step()
        torch.cuda.synchronize()
        for other in (second, third, fourth):
            assert all(torch.equal(a, b) for a, b in zip(first, other)), i


def test_rope_gradient_against_differences():
    n, h, d, sections = 12, 3, 16, [2, 3]
    q, k, g = rand((n, h, d), F32, 1), rand((n, 1, d), F32, 2), rand((n, h, d), F32, 3)
    pos, fr, w = torch.randint(0, 50, (n, 2)).int().cuda(), torch.rand(5).cuda(), rand((d,), F32, 4)
    leaves = [q.clone().requires_grad_(), w.clone().requires_grad_()]
    grads = torch.autograd.grad(at.qk_norm_rope(leaves[0], k, pos, fr, sections, leaves[1])[0], leaves, g)
    for i in range(2):
        x = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        f = []
        for e in (1e-5, -1e-5):
            a = [q.double().cpu(), w.double().cpu()]
            a[i] = a[i] + e * x
            f.append((oa.qk_norm_rope(a[0], pos, fr, sections, weight=a[1])["y"] * g.double().cpu()).sum())
        want = (f[0] - f[1]) / 2e-5
        assert abs((grads[i].double().cpu() * x).sum() - want) <= 1e-4 * (1 + abs(want))


def test_rope_refusals():
    q, k = rand((8, 4, 64), F16, 1), rand((8, 2, 64), F16, 2)
    pos, fr, w = torch.zeros(8, 1).int().cuda(), torch.ones(32).cuda(), torch.ones(64).cuda()
    ok = dict(q=q, k=k, positions=pos, inv_freq=fr, sections=[32])
    at.qk_norm_rope(**ok)
    for bad in (dict(k=k.float()), dict(k=k[:7]), dict(k=k[..., :32]), dict(q=q.double(), k=k.double()), dict(sections=[33]), dict(sections=[-1, 33]), dict(sections=[]), dict(sections=[31]),
                dict(sections=[8] * 5), dict(positions=pos[:7]), dict(positions=pos.double()), dict(positions=pos.cpu()), dict(positions=pos.expand(8, 2)), dict(inv_freq=fr[:31]),
                dict(inv_freq=fr.half()), dict(q_weight=w[:32]), dict(q_weight=w, k_weight=w.half()), dict(q_weight=w, normalize=False), dict(q_weight=w.double()), dict(eps=-1.0),
                dict(q=q[0]), dict(q=q.cpu()), dict(out=(q, q)), dict(out=(k, q)), dict(out=(q[:, :1].expand(-1, 4, -1), k))):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            at.qk_norm_rope(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="gradient"):
        at.qk_norm_rope(**{**ok, "q": q.clone().requires_grad_(), "out": (q, k)})
    a, b = at.qk_norm_rope(q[:0], k[:0], pos[:0], fr, [32], w)
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    leaf = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(at.qk_norm_rope(q[:0], k[:0], pos[:0], fr, [32], leaf)[0].sum(), leaf)
    assert not dw.any()                                                      # no tokens: a zero gradient, not a stale one


# ------------------------------------------------------------------------------------------------------------ used together
@pytest.mark.parametrize("block", [1, 48])
def test_a_block_over_keyframes(block):
    """projection, norm + rotation by (keyframe, row, column), attention, all gradients, against autograd in float64; then the same tokens
    keyframe by keyframe over a growing cache"""
    frames, h, w, heads, kv, d = 4, 6, 8, 4, 2, 32
    n, sections = frames * h * w, [4, 6, 6]
    x, wp = rand((n, 128), BF16, 1), rand((128, (heads + 2 * kv) * d), BF16, 2, 128 ** -0.5)
    at_ = torch.arange(n)
    pos = torch.stack([at_ // (h * w), at_ % (h * w) // w, at_ % w], 1).int().cuda()
    fr = torch.cat([100.0 ** (-torch.arange(s) / s) for s in sections]).float().cuda()
    wq, wk, g = rand((d,), F32, 3), rand((d,), F32, 4), rand((n, heads, d), BF16, 5)
    plan = at.PackedPlan([n], heads, kv, d, causal_block=block)
    qkv = (x @ wp).view(n, heads + 2 * kv, d).detach().requires_grad_()
    lw = [wq.clone().requires_grad_(), wk.clone().requires_grad_()]
    q, k = at.qk_norm_rope(qkv[:, :heads], qkv[:, heads:heads + kv], pos, fr, sections, *lw)
    o = at.packed_attention(q, k, qkv[:, heads + kv:], plan)
    grads = torch.autograd.grad(o, [qkv] + lw, g)

    t = [a.detach().double().cpu().requires_grad_() for a in (qkv, wq, wk)]
    ang = torch.cat([pos[:, i:i + 1].double().cpu() * f for i, f in enumerate(torch.split(fr.double().cpu(), sections))], 1)[:, None]
    turn = lambda z: torch.cat([z[..., :16] * ang.cos() - z[..., 16:] * ang.sin(), z[..., :16] * ang.sin() + z[..., 16:] * ang.cos()], -1)  # noqa: E731
    rms = lambda z, u: z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * u  # noqa: E731
    Q, K, V = turn(rms(t[0][:, :heads], t[1])), turn(rms(t[0][:, heads:heads + kv], t[2])), t[0][:, heads + kv:]
    K, V = (z.repeat_interleave(heads // kv, 1).transpose(0, 1) for z in (K, V))
    s = Q.transpose(0, 1) @ K.transpose(1, 2) / math.sqrt(d)
    s = s.masked_fill(torch.arange(n)[None] >= oa.keys_seen(n, n, block)[:, None], -math.inf)
    want_o = (s.softmax(-1) @ V).transpose(0, 1)
    want = torch.autograd.grad(want_o, t, g.double().cpu())
    # q and k are rounded between the two operators: half a step each, into scores of size up to |q| |k| / sqrt(d)
    u = oa.half_step(BF16)
    spread = (Q.detach().norm(dim=-1).max() * K.detach().norm(dim=-1).max() / math.sqrt(d)).item()
    rel = 2 * u * spread + 3 * u
    assert (o.double().cpu() - want_o.detach()).norm() <= rel * want_o.detach().norm()
    for a, b, name in zip(grads, want, ("qkv", "q_weight", "k_weight")):
        assert (a.double().cpu() - b).norm() <= 2 * rel * b.norm(), name

    if block == 48:                                                          # serving: a keyframe at a time over what is cached
        cache_k, cache_v = torch.zeros(n, kv, d, dtype=BF16, device="cuda"), torch.zeros(n, kv, d, dtype=BF16, device="cuda")
        with torch.no_grad():
            for f in range(frames):
                rows = slice(48 * f, 48 * f + 48)
                qn = torch.empty(48, heads, d, dtype=BF16, device="cuda")
                at.qk_norm_rope(qkv[rows, :heads], qkv[rows, heads:heads + kv], pos[rows].contiguous(), fr, sections, wq, wk, out=(qn, cache_k[rows]))
                cache_v[rows] = qkv[rows, heads + kv:]
                step = at.packed_attention(qn, cache_k, cache_v, at.PackedPlan([48], heads, kv, d, key_lengths=[48 * f + 48], causal_block=48))
                assert torch.equal(qn, q[rows]) and torch.equal(step, o[rows])
