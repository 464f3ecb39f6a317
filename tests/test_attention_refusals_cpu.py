"""Token operators without a GPU: what a call refuses before it writes anything."""
import ctypes
import os
import random
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "droid-slam_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

import droid_backends as db  # noqa: E402
from droid_amd import attention as at  # noqa: E402


def places(t):
    return torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()


@pytest.mark.parametrize("seed", range(8))
def test_views_that_share_memory_are_told_apart(seed):
    """against the elements themselves: strides alike and not, heads inside and outside rows, single rows and heads, broadcast ones"""
    rng = random.Random(seed)
    buf = torch.empty(4000, dtype=torch.float16)
    shared = apart = 0
    for _ in range(4000):
        d = rng.choice([2, 4, 8])
        st, sh = rng.choice([0, d, 3 * d, 4 * d, 37, 60]), rng.choice([0, d, 2 * d, 5 * d, 60])
        pair = []
        for _ in range(2):
            if rng.random() < 0.4:
                st, sh = rng.choice([d, 2 * d, 4 * d, 24, 61]), rng.choice([d, 2 * d, 30, 61])
            pair.append(buf.as_strided((rng.randint(0, 6), rng.randint(1, 5), d), (st, sh, 1), rng.randint(0, 150)))
        want = bool(set(places(pair[0])) & set(places(pair[1])))
        assert db._token_views_overlap(*pair) == db._token_views_overlap(*pair[::-1]) == want, [(t.shape, t.stride(), t.storage_offset()) for t in pair]
        for t in pair:
            assert db._token_view_overlaps_itself(t) == (len(set(places(t))) < t.numel())
        shared, apart = shared + want, apart + (not want)
    assert min(shared, apart) > 500


def test_heads_of_one_projection():
    """the layouts that out= meets: slices of one projection, caches, many rows"""
    qkv = torch.empty(100000, 12, 64, dtype=torch.float16)
    for a, b, want in ((qkv[:, :8], qkv[:, 2:10], True), (qkv[:, :8], qkv[:, 8:], False), (qkv[:, 0::2], qkv[:, 1::2], False), (qkv[:, 0::2], qkv[:, 0:1], True), (qkv[1:], qkv[:-1], True),
                       (qkv[:50000, :4], qkv[50000:], False), (qkv[::2], qkv[1::2], False), (qkv[:, :4, :32], qkv[:, :4, 32:], False), (qkv[:, :4, :32], qkv[:, 3:5, 16:48], True)):
        assert db._token_views_overlap(a, b) is want and not db._token_view_overlaps_itself(a)
    slots = torch.empty(2, 5000, 64, dtype=torch.float16).transpose(0, 1)   # heads outside rows
    assert db._token_views_overlap(slots[:100], slots[50:60]) and not db._token_views_overlap(slots[:100], slots[100:])
    assert db._token_views_overlap(qkv[:, :8], qkv.view(-1)[:12 * 100000 * 64 // 2].view(-1, 4, 64))       # (strides not alike, many rows: taken to overlap)


@pytest.mark.parametrize("wants_gradient", [False, True])
def test_forward_mode_is_refused(wants_gradient):
    """a tangent is not dropped in silence"""
    from torch.autograd import forward_ad as fw
    x, tangent = torch.zeros(4, 2, 32, dtype=torch.float16), torch.ones(4, 2, 32, dtype=torch.float16)
    plan = at.PackedPlan([4], 2, 2, 32, device="cpu")
    with fw.dual_level():
        dual = fw.make_dual(x.clone().requires_grad_() if wants_gradient else x, tangent)
        for a in ((dual, x, x), (x, dual, x), (x, x, dual)):
            with pytest.raises(RuntimeError, match="tangent"):
                at.packed_attention(*a, plan)
        for a in ((dual, x), (x, dual)):
            with pytest.raises(RuntimeError, match="tangent"):
                at.qk_norm_rope(*a, torch.arange(4), torch.ones(16), [16])


def test_gradients_that_nobody_forms_are_refused():
    """learned frequencies or positions would stay where they are in silence"""
    x, pos, fr = torch.zeros(4, 2, 32, dtype=torch.float16), torch.arange(4.0), torch.ones(16)
    for a in ((pos.clone().requires_grad_(), fr), (pos, fr.clone().requires_grad_())):
        for q in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="no gradient"):
                at.qk_norm_rope(q, x, *a, [16])
        with torch.no_grad(), pytest.raises(RuntimeError, match="device tensor"):
            at.qk_norm_rope(x, x, *a, [16])


def test_launches_of_too_many_threads_are_refused():
    """before anything is launched (there is no GPU here: a launch would come back as another code)"""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(db.__file__), "libdroid_hip.so"))
    i64, ptr, f32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    info = (i64 * 19)()

    def plan(rows, kv):
        return lib.dh_attn_plan((i64 * 1)(rows), (i64 * 1)(64), None, i64(1), kv, kv, 32, i64(0), None, i64(0), info)

    assert plan(128 * 500000, 32) == 0                                       # 1.6 10^7 workgroups of 256
    assert plan(128 * 600000, 32) == 1
    sec, t = (ctypes.c_int * 1)(1), (ptr(256), i64(512), i64(256))

    def rope(tokens, dim):
        return lib.dh_qk_norm_rope_fwd(*t, *t, *t, *t, ptr(256), 0, ptr(256), sec, 1, ptr(0), ptr(0), 1, 0, i64(tokens), 1, 0, dim, 0, f32(1e-6), 1, ptr(0))

    assert rope(2 ** 29 + 1, 256) == 1 and rope(2 ** 32 + 1, 2) == 1
