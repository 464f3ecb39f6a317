"""Token operators on the GPU at the ends of their range: results against the definition, within bounds that follow from the roundings."""
import ctypes
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
from tests.test_attention_gpu import BF16, F16, inputs, near, rand  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("size", [25, 200, 1000])
def test_gradients_whose_factors_are_larger_than_fp16(d, size):
    """two keys of equal weight and opposite values under a large gradient: dS = +-d size / 2 is past fp16's numbers (lifted by 2^4 past them even
    sooner), every gradient is inside them"""
    q, k, v = torch.zeros(3, 2, d), rand((2, 1, d), F16, 1, 0.25).cpu().float(), torch.ones(2, 1, d)
    q[..., 1], k[:, :, 1], v[1] = 3.0, 0.5, -1.0                             # equal scores: weights of one half
    g = torch.full((3, 2, d), float(size)) * torch.tensor([1.0, -1.0, 0.001]).view(3, 1, 1)
    q, k, v, g = (t.half().cuda() for t in (q, k, v, g))
    r = oa.attention(q, k, v, [3], [2], grad=g)
    assert max(r[n].abs().max() for n in ("dq", "dk", "dv")) < 65504
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = at.packed_attention(*leaves, at.PackedPlan([3], 2, 1, d, key_lengths=[2]))
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("lengths,keys,heads,kv,d,block,size", [([300, 40], None, 4, 2, 64, 1, 2000.0), ([150], None, 4, 2, 128, 0, 8000.0), ([200], None, 2, 2, 32, 10, 2000.0),
                                                                ([2, 3], [9000, 5000], 8, 2, 64, 0, 8000.0), ([9000], [9], 3, 1, 64, 0, 50.0)])
def test_gradients_under_a_loss_scale(lengths, keys, heads, kv, d, block, size):
    """gradients of thousands in some rows and ordinary ones in others (walks that are split among them)"""
    q, k, v, g = inputs(lengths, keys, heads, kv, d, F16, 90)
    q, k = q * 0.5, k * 0.25
    g[::3] *= size
    r = oa.attention(q, k, v, lengths, keys, block=block, grad=g)
    assert max(r[n].abs().max() for n in ("dq", "dk", "dv")) < 65504
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = at.packed_attention(*leaves, at.PackedPlan(lengths, heads, kv, d, key_lengths=keys, causal_block=block))
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, g)):
        near(t, r[n], r[n + "_err"], n)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("a,b", [(4, 4), (64, 64), (128, 128), (512, 256), (2048, 1536), (4096, 1536), (4096, 2816)])
@pytest.mark.parametrize("d,lengths,keys,heads", [(64, [3, 40], [4, 4], 2), (128, [5], [8], 1), (32, [1, 1], [8192, 2048], 8), (128, [2, 1], [16384, 8], 4), (64, [7000], [4], 8)])
def test_gradients_at_large_scores(d, lengths, keys, heads, a, b, sign, dtype):
    """all keys are alike, so that each weighs 1 / keys whatever the score is: +- a b sqrt(d), up to 9 10^7.  Lengths are powers of two: the weights
    are exact in 16 bits, dV is a mean of dO, dQ and dK are what 32-bit sums leave of zero"""
    m, l = sum(lengths), sum(keys)
    scale = 64 ** 0.5 / d                                                    # scores of a b 8 for every d
    q = torch.full((m, heads, d), float(a), dtype=dtype, device="cuda")
    k = torch.full((l, 1, d), float(sign * b), dtype=dtype, device="cuda")
    v, g = rand((1, 1, d), dtype, 1).expand(l, 1, d).contiguous(), rand((m, heads, d), dtype, 2)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = at.packed_attention(*leaves, at.PackedPlan(lengths, heads, 1, d, key_lengths=keys), scale=scale, return_lse=True)
    assert torch.equal(o, v[:1].expand(m, heads, d))                         # a mean of equal numbers
    dq, dk, dv = (t.double().cpu() for t in torch.autograd.grad(o, leaves, g))
    u, u32 = oa.half_step(dtype), 2.0 ** -24
    G, V = g.double().cpu(), v.double().cpu()
    q0 = k0 = 0
    for x, y in zip(lengths, keys):
        # dP and delta are sums of d products each that start alike; delta once more
        dS = 4 * (d + 8) * u32 * (G[q0:q0 + x].abs() * V[0].abs()).sum(-1).max() / y
        want, size = G[q0:q0 + x].sum((0, 1)) / y, G[q0:q0 + x].abs().sum((0, 1)) / y
        err = u * want.abs() + (x * heads + 64) * u32 * size + 2.0 ** -25 + 2.0 ** -28 * size * y
        assert ((dv[k0:k0 + y, 0] - want).abs() <= err).all(), "dv: %g" % (dv[k0:k0 + y, 0] - want).abs().max()
        assert dq[q0:q0 + x].abs().max() <= (dS + 2.0 ** -28) * y * scale * b * (1 + u), "dq"
        assert dk[k0:k0 + y].abs().max() <= (dS + 2.0 ** -28) * x * heads * scale * a * (1 + u), "dk"
        q0, k0 = q0 + x, k0 + y


def test_out_over_slices_of_one_buffer():
    """an out= that shares memory with an input is refused, however the views lie; beside them it may lie in the same buffer"""
    n, d = 300, 64
    qkv = rand((n, 24, d), F16, 1)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:12]
    plan = at.PackedPlan([n], 8, 2, d, causal_block=1)
    want = at.packed_attention(q, k, v, plan)
    keep = qkv.clone()
    for out in (q, qkv[:, 2:10], qkv[:, 10:18], qkv[:, 4:20:2], qkv.view(-1)[8 * d:][:n * 8 * d].view(n, 8, d), qkv.as_strided((n, 8, d), (24 * d, 32, 1), 14 * d),
                qkv.as_strided((n, 8, d), (0, d, 1), 0), qkv.as_strided((n, 8, d), (8, 24 * d, 1), 14 * d)):
        with pytest.raises(RuntimeError, match="overlaps|same place"):
            at.packed_attention(q, k, v, plan, out=out)
    pos, fr = torch.arange(n, device="cuda"), torch.rand(32, device="cuda")
    for out in ((qkv[:, 1:9], qkv[:, 12:14]), (qkv[:, 12:20], qkv[:, 9:11]), (qkv[:, 12:20], qkv[:, 19:21]), (qkv[:, 8:16], qkv[:, 16:18]), (qkv[:, 12:20], qkv[:, 6:8]), (q, qkv[:, 7:9])):
        with pytest.raises(RuntimeError, match="overlaps"):
            at.qk_norm_rope(q, k, pos, fr, [32], out=out)
    assert torch.equal(qkv, keep)                                            # nothing was written
    for out in (qkv[:, 12:20], qkv[:, 13:21]):
        assert torch.equal(at.packed_attention(q, k, v, plan, out=out), want)
    turned = [t.clone() for t in at.qk_norm_rope(q, k, pos, fr, [32])]
    for out in ((qkv[:, 12:20], qkv[:, 20:22]), (q, k)):
        got = at.qk_norm_rope(q, k, pos, fr, [32], out=out)
        assert torch.equal(got[0], turned[0]) and torch.equal(got[1], turned[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("low", [-16.0, -17.40625, -18.5])
def test_a_long_tail_of_small_weights(low, d, dtype):
    """one key far above thousands of others: their weights are small one by one and count together (walks that are not split)"""
    heads, n, rows = 8, 8192, 8960
    q, k, v = torch.zeros(rows, heads, d, dtype=dtype), torch.zeros(n, heads, d, dtype=dtype), torch.ones(n, heads, d, dtype=dtype)
    q[..., 0], k[1:, :, 0], v[0] = 1.0, low, 0.0
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    plan = at.PackedPlan([rows], heads, heads, d, key_lengths=[n])
    assert int(plan.info[7]) == 0                                            # (no joins)
    o, lse = at.packed_attention(q, k, v, plan, scale=1.0, return_lse=True)
    r = oa.attention(q[:1, :1], k[:, :1], v[:, :1], [1], [n], scale=1.0)
    assert bool((o == o[:1, :1]).all()) and bool((lse == lse[:1, :1]).all())
    near(o[:1, :1], r["o"], r["o_err"], "o")
    near(lse[:1, :1], r["lse"], r["lse_err"], "lse")


@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_of_32_bit_features(interleaved):
    """(1, 0) turns into (cos, sin): nothing is rounded but the sine and the cosine themselves, by half a step"""
    n, d = 20000, 64
    x = torch.zeros(n, 1, d, device="cuda")
    x[..., 0:d:2 if interleaved else 1][..., :d // 2] = 1.0
    if not interleaved:
        x[..., d // 2:] = 0.0
    pos = torch.randint(-3000000, 3000000, (n,), generator=torch.Generator().manual_seed(1)).cuda()
    pos[:3000] = torch.arange(3000, device="cuda")
    fr = (10000.0 ** (-torch.arange(d // 2) / (d // 2))).float().cuda()
    y, _ = at.qk_norm_rope(x, x[:, :0], pos, fr, [d // 2], normalize=False, interleaved=interleaved)
    ang = pos.double()[:, None] * fr.double()
    c, s = (y[:, 0, 0::2], y[:, 0, 1::2]) if interleaved else (y[:, 0, :d // 2], y[:, 0, d // 2:])
    for got, want in ((c, ang.cos()), (s, ang.sin())):
        # a position times a frequency keeps 53 bits: 3 10^6 2^-52 beside the half step
        assert bool(((got.double() - want).abs() <= 2.0 ** -24 * want.abs() + 3e6 * 2.0 ** -51).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,keys", [([5], [5]), ([1, 3], [9000, 3])])
def test_rows_whose_scores_are_all_minus_infinity(lengths, keys, dtype):
    """keys of -inf under positive queries: there is no softmax of that, in a split row neither; others do not change"""
    q, k, v, _ = inputs(lengths, keys, 2, 1, 64, dtype, 3)
    q = q.abs()
    if keys[0] == 5:
        k[0] = -float("inf")                                                 # token 0 sees only this key
        o, lse = at.packed_attention(q, k, v, at.PackedPlan(lengths, 2, 1, 64, causal_block=1), return_lse=True)
        assert bool(o[0].isnan().all()) and bool(torch.isfinite(o[1:]).all())
    else:
        k[:9000] = -float("inf")
        o, lse = at.packed_attention(q, k, v, at.PackedPlan(lengths, 2, 1, 64, key_lengths=keys), return_lse=True)
        assert bool(o[0].isnan().all()) and bool(torch.isfinite(o[1:]).all())
    assert bool((lse[0] == -float("inf")).all())


def test_capture_beside_a_living_graph_of_a_sliced_leaf_is_refused():
    """heads sliced from one leaf, and what is computed from a leaf before the call: the accumulator lives on the eager stream, autograd would end the process"""
    n, d = 40, 64
    qkv, g = rand((n, 8, d), BF16, 1).requires_grad_(), rand((n, 4, d), BF16, 2)
    w = torch.ones(d, device="cuda", requires_grad=True)
    plan = at.PackedPlan([n], 4, 2, d, causal_block=1)
    pos, fr = torch.arange(n, device="cuda", dtype=torch.int32), torch.rand(32, device="cuda")

    def step(x, u):
        q, k = at.qk_norm_rope(x[:, :4], x[:, 4:6], pos, fr, [32], u, u)
        return at.packed_attention(q, k, x[:, 6:], plan)

    alive = step(qkv, w * 2)
    for call in (lambda: at.packed_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], plan), lambda: at.qk_norm_rope(qkv.detach()[:, :4], qkv.detach()[:, 4:6], pos, fr, [32], w * 2),
                 lambda: at.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], pos, fr, [32]), lambda: step(qkv * 1, w)):
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    want = torch.autograd.grad(alive, (qkv, w), g)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(step(qkv, w * 2), (qkv, w), g)
    for _ in range(3):
        graph.replay()
        step(qkv.detach(), w.detach() * 2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad as fw
    x, w, pos, fr = rand((8, 2, 64), F16, 1), torch.ones(64, device="cuda"), torch.arange(8.0, device="cuda"), torch.ones(32, device="cuda")
    plan = at.PackedPlan([8], 2, 2, 64)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: at.packed_attention(x, x, dual(x), plan), lambda: at.packed_attention(dual(x.clone().requires_grad_()), x, x, plan),
                     lambda: at.qk_norm_rope(x, x, pos, fr, [32], dual(w)), lambda: at.qk_norm_rope(x, x, dual(pos), fr, [32]), lambda: at.qk_norm_rope(x, x, pos, dual(fr), [32])):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert at.packed_attention(x, x, x, plan).shape == x.shape


def test_out_is_seen_by_autograd():
    """what is written through out= is a new value: a backward pass that kept the old one says so; an out= that wants a gradient itself is refused"""
    n, d = 20, 64
    q, k, v, g = inputs([n], None, 4, 2, d, F16, 7)
    pos, fr, plan = torch.arange(n, device="cuda"), torch.rand(32, device="cuda"), at.PackedPlan([n], 4, 2, d)
    a, w = torch.ones_like(q).requires_grad_(), torch.ones_like(k).requires_grad_()
    kept = [(a * q).sum(), (w * k).sum()]
    with torch.no_grad():
        at.qk_norm_rope(q, k, pos, fr, [32], out=(q, k))
    for t in kept:
        with pytest.raises(RuntimeError, match="inplace"):
            t.backward()
    buf = torch.zeros(n, 8, d, dtype=F16, device="cuda")
    kept = (torch.ones_like(buf).requires_grad_() * buf).sum()
    with torch.no_grad():
        at.packed_attention(q, k, v, plan, out=buf[:, 2:6])                  # (a view: the whole buffer is another one)
    with pytest.raises(RuntimeError, match="inplace"):
        kept.backward()
    leaf = torch.zeros_like(q).requires_grad_()
    for call in (lambda: at.packed_attention(q, k, v, plan, out=leaf), lambda: at.qk_norm_rope(q, k, pos, fr, [32], out=(leaf, torch.empty_like(k)))):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with torch.inference_mode():
        out = torch.empty_like(q)
        assert torch.equal(at.packed_attention(q, k, v, plan, out=out), at.packed_attention(q, k, v, plan))


def test_a_plan_with_another_plans_info_stays_inside_the_workspace():
    """as many items, other lengths: what reaches behind the rows of the info is left out, forward and backward, whatever rows the tensors have"""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(at.droid_backends.__file__), "libdroid_hip.so"))
    i64, ptr, f32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    lib.dh_attn_bwd_workspace_bytes.restype = ctypes.c_size_t
    h, kv, d, rows = 4, 2, 64, 40
    q, k, v, g = inputs([rows], None, h, kv, d, F16, 5)
    info, other = (i64 * 19)(), (i64 * 19)()
    items = (ctypes.c_int32 * 24)()
    one = lambda n: (i64 * 1)(n)  # noqa: E731
    assert lib.dh_attn_plan(one(8), one(8), None, i64(1), h, kv, d, i64(0), None, i64(0), info) == 0
    assert lib.dh_attn_plan(one(31), one(31), None, i64(1), h, kv, d, i64(0), items, i64(24), other) == 0 and info[0] == other[0] == 24
    items = torch.frombuffer(items, dtype=torch.int32).clone().cuda()
    n = lib.dh_attn_bwd_workspace_bytes(info)
    ws = torch.full((n // 4 + 4096,), 7.0, device="cuda")
    o, dq, lse = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full((rows, h), 7.0, device="cuda")
    dk, dv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    t = lambda x: (ptr(x.data_ptr()), i64(x.stride(0)), i64(x.stride(1)))  # noqa: E731
    p = lambda x: ptr(x.data_ptr())  # noqa: E731
    tail = (p(items), info, 0, i64(rows), i64(rows), f32(0.125), 0, p(ws), ctypes.c_size_t(n), ptr(torch.cuda.current_stream().cuda_stream))
    assert lib.dh_attn_fwd(*t(q), *t(k), *t(v), *t(o), ptr(0), p(lse), *tail) == 0
    assert lib.dh_attn_bwd(*t(g), *t(q), *t(k), *t(v), *t(o), ptr(0), p(lse), *t(dq), *t(dk), *t(dv), *tail) == 0
    torch.cuda.synchronize()
    assert all(bool((x == 7).all()) for x in (o, lse, dq, dk, dv, ws[n // 4:]))
