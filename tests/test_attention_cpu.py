"""Token operators without a GPU: the plan of packed attention, the refusals of every entry point, the oracle against differences."""
import ctypes
import itertools
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "droid-slam_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

import droid_backends as db  # noqa: E402
from droid_amd import attention as at  # noqa: E402
from oracle import attention as oa  # noqa: E402

FIELDS = ["ints", "heads", "kv_heads", "head_dim", "causal_block", "waves", "n_fwd", "n_join", "n_dq", "n_dq_join", "n_dkv", "n_dkv_join", "n_slots", "n_dq_slots", "n_dkv_slots",
          "q_rows", "k_rows", "k_total", "keys_shared"]


def plan(lengths, heads, kv_heads, dim, **kw):
    p = at.PackedPlan(lengths, heads, kv_heads, dim, device="cpu", **kw)
    info = dict(zip(FIELDS, p.info.tolist()))
    items = p.items.view(-1, 8).tolist()
    cut = list(itertools.accumulate([0] + [info[n] for n in ("n_fwd", "n_join", "n_dq", "n_dq_join", "n_dkv", "n_dkv_join")]))
    return info, [items[a:b] for a, b in zip(cut, cut[1:])]


PLANS = [([1], None, 1, 1, 0), ([48], None, 4, 4, 0), ([5, 0, 300, 1], None, 8, 2, 1), ([5, 0, 300, 1], [700, 3, 0, 1], 6, 2, 1), ([130, 17], [64, 4000], 32, 1, 100),
         ([1] * 9, [1, 0, 63, 64, 65, 5000, 9000, 129, 20000], 16, 2, 1), ([2000], [500], 4, 4, 7), ([700], [9000], 3, 1, 0), ([9000], [40], 8, 1, 0), ([6000], None, 16, 2, 100), ([], None, 4, 2, 0)]


@pytest.mark.parametrize("dim,keys_a_tile", [(64, 64), (128, 128)])
@pytest.mark.parametrize("lengths,key_lengths,heads,kv_heads,block", PLANS)
def test_plan_covers_every_row_and_key_once(lengths, key_lengths, heads, kv_heads, block, dim, keys_a_tile):
    """each visible (row, key) pair is in exactly one forward item, one dQ item and one dK / dV item"""
    keys = lengths if key_lengths is None else key_lengths
    info, (fwd, join, dq, dq_join, dkv, dkv_join) = plan(lengths, heads, kv_heads, dim, key_lengths=key_lengths, causal_block=block)
    assert info["q_rows"] == sum(lengths) and info["k_rows"] == sum(keys) == info["k_total"] and not info["keys_shared"]
    group = heads // kv_heads
    q0 = k0 = 0
    for m, l in zip(lengths, keys):
        seen = torch.arange(l)[None] < oa.keys_seen(m, l, block)[:, None]
        for items, tokens in ((fwd, info["waves"] * 32 // group), (dq, 128 // group)):
            hit, rows = torch.zeros(m, l, dtype=torch.int), torch.zeros(m, dtype=torch.int)
            for qs, ql, ks, kl, first, begin, end, slot in items:
                if (qs, ql) != (q0, m) or (ks, kl) != (k0, l) or m == 0:
                    continue
                assert begin % 64 == 0 and (end % 64 == 0 or end == int(oa.keys_seen(m, l, block)[min(m, first + tokens) - 1]) or end <= l)
                hit[first:first + tokens, begin:end] += 1
                rows[first:first + tokens] += begin == 0
            assert bool((hit[seen] == 1).all()) and bool((hit <= 1).all()) and bool((rows == 1).all())
        hit = torch.zeros(m, l, dtype=torch.int)
        for qs, ql, ks, kl, first, begin, end, _ in dkv:
            if (qs, ql) == (q0, m) and (ks, kl) == (k0, l) and l:
                assert 0 <= begin <= end <= m
                hit[begin:end, first:first + keys_a_tile] += 1
        assert bool((hit[seen] == 1).all()) and bool((hit <= 1).all())
        q0, k0 = q0 + m, k0 + l
    for items, joins, n in ((fwd, join, "n_slots"), (dq, dq_join, "n_dq_slots"), (dkv, dkv_join, "n_dkv_slots")):
        slots = sorted(x for j in joins for x in range(j[5], j[5] + j[6]))
        assert slots == list(range(info[n])) == sorted(i[7] for i in items if i[7] >= 0)


def test_plan_of_shared_keys_and_gaps():
    info, _ = plan([4, 4], 2, 2, 32, key_lengths=[10, 10], key_starts=[0, 5])
    assert info["keys_shared"] == 1 and info["k_rows"] == 15 and info["k_total"] == 20
    info, _ = plan([4, 4], 2, 2, 32, key_lengths=[10, 10], key_starts=[100, 20])
    assert info["keys_shared"] == 0 and info["k_rows"] == 110 and info["k_total"] == 20
    info, _ = plan([4, 4], 2, 2, 32, key_lengths=[0, 10], key_starts=[25, 20])
    assert info["keys_shared"] == 0


@pytest.mark.parametrize("kw", [dict(lengths=[-1]), dict(lengths=[4], key_lengths=[-2]), dict(lengths=[4], key_lengths=[4, 4]), dict(lengths=[4], key_starts=[-1]),
                                dict(lengths=[2 ** 31]), dict(lengths=[2 ** 30, 2 ** 30]), dict(lengths=[4], heads=3, kv_heads=2), dict(lengths=[4], heads=64, kv_heads=1),
                                dict(lengths=[4], kv_heads=0), dict(lengths=[4], head_dim=12), dict(lengths=[4], head_dim=136), dict(lengths=[4], head_dim=0),
                                dict(lengths=[4], causal_block=-1)])
def test_plan_refuses(kw):
    a = dict(heads=4, kv_heads=4, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises((RuntimeError, TypeError)):
        at.PackedPlan(**a)


def test_cpu_tensors_are_refused():
    p = at.PackedPlan([4], 2, 2, 32, device="cpu")
    x = torch.zeros(4, 2, 32, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="device tensor"):
        at.packed_attention(x, x, x, p)
    with pytest.raises(RuntimeError, match="device tensor"):
        at.qk_norm_rope(x, x, torch.zeros(4, 1, dtype=torch.int32), torch.ones(16), [16])


def test_c_entries_refuse_before_a_launch():
    """bad arguments and buffers come back as codes; no pointer is looked at"""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(db.__file__), "libdroid_hip.so"))
    lib.dh_attn_fwd_workspace_bytes.restype = lib.dh_attn_bwd_workspace_bytes.restype = lib.dh_qk_norm_rope_bwd_workspace_bytes.restype = ctypes.c_size_t
    i64, ptr = ctypes.c_int64, ctypes.c_void_p
    info = (i64 * len(FIELDS))()

    def make(lengths, keys, starts=None, heads=4, kv=2, dim=64, block=1, room=None):
        arr = lambda v: None if v is None else (i64 * max(1, len(v)))(*v)  # noqa: E731
        buf = None if room is None else (ctypes.c_int32 * max(1, room))()
        return lib.dh_attn_plan(arr(lengths), arr(keys), arr(starts), i64(len(lengths)), heads, kv, dim, i64(block), buf, i64(room or 0), info)

    assert make([5], [9]) == 0 and info[0] == 8 * sum(info[6:12])
    assert make([5], [9], room=info[0] - 1) == 2                             # too small a buffer: nothing is written behind it
    assert make([5], [9], room=int(info[0])) == 0
    assert make([-1], [9]) == 1 and make([5], [9], starts=[-3]) == 1 and make([5], [9], dim=20) == 1 and make([5], [9], heads=5) == 1 and make([5], [9], block=-1) == 1

    def fwd(q=256, k=256, v=256, o=256, low=0, lse=256, plan=256, dtype=0, rows=5, keys=9, scale=0.1, st=(256, 64), ws=0, wsb=0, info=info):
        t = lambda p: (ptr(p), i64(st[0]), i64(st[1]))  # noqa: E731
        return lib.dh_attn_fwd(*t(q), *t(k), *t(v), *t(o), ptr(low), ptr(lse), ptr(plan), info, dtype, i64(rows), i64(keys), ctypes.c_float(scale), 0, ptr(ws), ctypes.c_size_t(wsb), ptr(0))

    make([5], [9])
    for bad in (dict(q=0), dict(q=8), dict(k=0), dict(v=264), dict(o=0), dict(low=8), dict(lse=0), dict(plan=0), dict(dtype=1), dict(dtype=2), dict(rows=4), dict(keys=8), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(st=(252, 64)), dict(st=(-256, 64)), dict(st=(1 << 25, 64)), dict(st=(256, 1 << 26)), dict(info=None)):
        assert fwd(**bad) == 1, bad
    assert make([1], [100000], heads=8, kv=1) == 0 and info[12] > 0 and lib.dh_attn_fwd_workspace_bytes(info) > 0
    assert fwd(rows=1, keys=100000) == 2                                     # split rows need the workspace

    def bwd(ws=256, wsb=1 << 20, dtype=0, rows=5, keys=9, dq=256, dk=256, plan=256, lse=256):
        t = lambda p: (ptr(p), i64(256), i64(64))  # noqa: E731
        return lib.dh_attn_bwd(*t(256), *t(256), *t(256), *t(256), *t(256), ptr(0), ptr(lse), *t(dq), *t(dk), *t(256), ptr(plan), info, dtype, i64(rows), i64(keys), ctypes.c_float(0.1), 0,
                               ptr(ws), ctypes.c_size_t(wsb), ptr(0))

    make([5], [9])
    assert bwd(ws=0) == 2 and bwd(wsb=8) == 2 and bwd(dtype=1) == 1 and bwd(rows=4) == 1 and bwd(keys=2) == 1 and bwd(dq=0) == 1 and bwd(dk=8) == 1 and bwd(plan=0) == 1 and bwd(lse=0) == 1
    make([5, 5], [9, 9], starts=[0, 3])
    assert bwd(rows=10, keys=12) == 1                                        # shared keys

    sec = (ctypes.c_int * 4)(4, 6, 6, 0)

    def rope(q=256, qo=256, pos=256, pt=0, fr=256, sections=sec, axes=3, qw=0, wt=1, dtype=0, tokens=3, heads=2, kv=2, dim=32, norm=1, eps=1e-6, st=(64, 32)):
        t = lambda p: (ptr(p), i64(st[0]), i64(st[1]))  # noqa: E731
        return lib.dh_qk_norm_rope_fwd(*t(q), *t(256), *t(qo), *t(256), ptr(pos), pt, ptr(fr), sections, axes, ptr(qw), ptr(0), wt, dtype, i64(tokens), heads, kv, dim, norm,
                                       ctypes.c_float(eps), 0, ptr(0))

    for bad in (dict(q=0), dict(q=257), dict(qo=0), dict(pos=0), dict(pt=3), dict(fr=0), dict(sections=None), dict(axes=0), dict(axes=5), dict(wt=2), dict(dtype=2), dict(tokens=-1),
                dict(heads=-1), dict(dim=33), dict(dim=0), dict(dim=258), dict(dim=30), dict(eps=-1.0), dict(eps=float("nan")), dict(st=(-64, 32)), dict(qw=256, norm=0),
                dict(sections=(ctypes.c_int * 4)(-1, 6, 6, 0)), dict(sections=(ctypes.c_int * 4)(6, 6, 6, 0))):
        assert rope(**bad) == 1, bad
    assert rope(dim=254, sections=(ctypes.c_int * 4)(1, 0, 0, 0), st=(512, 256)) == 4                  # above 128 channels in single channels a lane
    assert rope(tokens=0, q=0, qo=0) == 0
    assert lib.dh_qk_norm_rope_bwd_workspace_bytes(0) == 0 and lib.dh_qk_norm_rope_bwd_workspace_bytes(64) > 0


def test_oracle_gradients_against_differences():
    """the float64 formulas that the GPU tests compare with, against central differences of their own forward"""
    torch.manual_seed(0)
    lengths, keys, heads, kv, d = [3, 5, 2], [6, 4, 0], 4, 2, 8
    t = {"q": torch.randn(10, heads, d, dtype=torch.float64), "k": torch.randn(10, kv, d, dtype=torch.float64), "v": torch.randn(10, kv, d, dtype=torch.float64)}
    g = torch.randn(10, heads, d, dtype=torch.float64)
    for block in (0, 1, 3):
        r = oa.attention(t["q"], t["k"], t["v"], lengths, keys, block=block, grad=g)
        for n in "qkv":
            x = torch.randn_like(t[n])
            f = [(oa.attention(**{**t, n: t[n] + h * x}, lengths=lengths, key_lengths=keys, block=block)["o"] * g).sum() for h in (1e-5, -1e-5)]
            assert abs((f[0] - f[1]) / 2e-5 - (r["d" + n] * x).sum()) < 1e-7
    x, w, g = torch.randn(7, 3, 12, dtype=torch.float64), torch.randn(12, dtype=torch.float64), torch.randn(7, 3, 12, dtype=torch.float64)
    pos, fr = torch.randint(-9, 9, (7, 2)), torch.rand(4)
    for inter, norm in itertools.product((False, True), (False, True)):
        a = dict(positions=pos, inv_freq=fr, sections=[1, 3], normalize=norm, interleaved=inter)
        r = oa.qk_norm_rope(x, weight=w if norm else None, grad=g, **a)
        dx, dw = torch.randn_like(x), torch.randn_like(w)
        f = [(oa.qk_norm_rope(x + h * dx, weight=w if norm else None, **a)["y"] * g).sum() for h in (1e-5, -1e-5)]
        assert abs((f[0] - f[1]) / 2e-5 - (r["dx"] * dx).sum()) < 1e-7
        if norm:
            f = [(oa.qk_norm_rope(x, weight=w + h * dw, **a)["y"] * g).sum() for h in (1e-5, -1e-5)]
            assert abs((f[0] - f[1]) / 2e-5 - (r["dw"] * dw).sum()) < 1e-7
