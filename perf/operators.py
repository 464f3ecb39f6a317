"""The token operators of droid_amd.attention, as they are measured.

A keyframe's feature map is a grid of tokens; a window of keyframes is a packed sequence of them (frame by frame, row by row), several
windows are packed one behind the other.  Two operators, each with its backward pass:

  rope   norm of every query and key head, and the rotation by the token's position along one to three axes (keyframe, row, column),
         in one pass
  attn   softmax attention over packed sequences of different lengths with grouped heads: every key, the keys up to the token, or the
         keys up to the end of the token's keyframe; as many queries as keys, or a few new queries over a long window

`own` False computes them from elementary torch operations in 32 bits; `own` True calls the framework."""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
BASE = 10000.0


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "droid-slam_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from droid_amd import attention
    return attention


def _ints(text):
    return [int(x) for x in text.split(",")]


# ---------------------------------------------------------------------------------------------------------------- the cases
def _rope(name, dtype, tokens, heads, kv_heads, dim, sections, height, width, normalize=True, interleaved=False, train=False):
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "sections": sections,
            "height": height, "width": width, "normalize": normalize, "interleaved": interleaved, "train": train}


def _attn(name, dtype, q_lens, heads, kv_heads, dim, block, k_lens="", pad=0, train=False):
    """`block`: 0 every key, 1 the keys up to the token, n the keys up to the end of the token's keyframe of n tokens"""
    return {"name": name, "op": "attn", "dtype": dtype, "q_lens": q_lens, "k_lens": k_lens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "block": block, "pad": pad, "train": train}


def listed():
    return [
        # one new keyframe on the coarsest grid of a 48x64 feature map (6x8): the frontend adds keyframes one at a time, latency is all
        _rope("rope_one_keyframe", "f16", 48, 4, 4, 32, "4,6,6", 6, 8),
        # an odd grid (41x73 features of a 16:9 video), three keyframes, 32-bit features, rotation alone, pairs side by side
        _rope("rope_odd_grid", "f32", 3 * 41 * 73, 6, 6, 40, "4,8,8", 41, 73, normalize=False, interleaved=True),
        # the frontend's window of 25 keyframes of 30x40 tokens with grouped heads: bound by memory
        _rope("rope_window", "bf16", 25 * 1200, 16, 4, 128, "16,24,24", 30, 40),
        # training steps: a short clip of seven keyframes at 24x32, and the whole window
        _rope("rope_train_clip", "f16", 7 * 768, 8, 8, 64, "8,12,12", 24, 32, train=True),
        _rope("rope_train_window", "bf16", 25 * 1200, 16, 4, 128, "16,24,24", 30, 40, train=True),
        # one new keyframe over itself: the smallest call
        _attn("attn_one_keyframe", "f16", "48", 4, 4, 32, 0),
        # serving: one query for each of 32 videos over windows of very different lengths (one key to 27 keyframes of 30x40), grouped heads
        _attn("attn_single_queries", "bf16", ",".join(["1"] * 32), 16, 2, 128, 1,
              ",".join(str(n) for n in (1, 17, 48, 192, 333, 768, 1200, 1201, 2400, 2993, 3600, 4800, 5376, 6001, 7200, 8979, 9600, 10800, 12000, 13200, 14400,
                                        15600, 16800, 18000, 19200, 20400, 21600, 22800, 24000, 25200, 30000, 32400))),
        # a new keyframe of 24x32 tokens over a window of 30 keyframes, itself included
        _attn("attn_new_keyframe_over_window", "f16", "768", 8, 8, 64, 768, str(30 * 768)),
        # clips of different lengths packed, token by token, rows of padding behind them
        _attn("attn_packed_clips", "bf16", "5376,48,2993,1,768,192,4095,1344,0,2017", 8, 4, 64, 1, pad=61),
        # sixteen keyframes of 30x40 over each other, keyframe by keyframe
        _attn("attn_window", "bf16", str(16 * 1200), 16, 4, 128, 1200),
        # training steps: packed clips; a window of twelve keyframes
        _attn("attn_train_clips", "f16", "2304,192,1501,48,2993,768,1", 8, 8, 64, 192, pad=7, train=True),
        _attn("attn_train_window", "bf16", str(12 * 1200), 16, 4, 128, 1200, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16"])
    train = rng.random() < 0.5
    if rng.random() < 0.45:
        dtype = rng.choice(["f16", "bf16", "f32"])
        dim = rng.choice([16, 32, 40, 64, 80, 96, 128])
        axes = rng.randint(1, 3)
        pairs = dim // 2 if rng.random() < 0.7 else dim // 4
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 4])
        high = max(64, min(30000, 30000 * 20 * 128 * 2 // ((heads + kv) * dim * (4 if dtype == "f32" else 2))))
        height, width = rng.randint(3, 41), rng.randint(3, 73)
        return _rope_case(dtype, _log(rng, 1, high), heads, kv, dim, sections, height, width, rng.random() < 0.7, rng.random() < 0.4, train)
    dim = rng.choice([32, 64, 64, 128, 128, 40, 80, 96])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    seqs = _log(rng, 1, 16)
    few = rng.random() < 0.3
    longest = _log(rng, 8, 32000 if few else 8000)
    while seqs * heads * dim * longest * (16 if few else longest) * (3.5 if train else 1) > 14400 ** 2 * 16 * 128:
        longest = max(8, int(longest * 0.8))
    k_lens = [rng.randint(0, longest) for _ in range(seqs)]
    whole = rng.randrange(seqs)
    k_lens[whole] = longest
    if few:
        q_lens = [rng.randint(0, 16) for _ in k_lens]
    elif rng.random() < 0.7:
        q_lens = list(k_lens)
    else:
        q_lens = [rng.randint(0, longest) for _ in k_lens]
    q_lens[whole] = max(1, q_lens[whole])                        # one query at least that sees several keys
    block = rng.choice([0, 1, 1, rng.randint(2, 1200)])
    text = lambda v: ",".join(str(n) for n in v)  # noqa: E731
    c = _attn("", dtype, text(q_lens), heads, kv, dim, block, "" if q_lens == k_lens else text(k_lens), rng.choice([0, 0, rng.randint(1, 100)]), train)
    del c["name"]
    return c


def _rope_case(*args):
    c = _rope("", *args)
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------------------------- the inputs
def _lengths(case):
    q = _ints(case["q_lens"])
    return q, (_ints(case["k_lens"]) if case["k_lens"] else list(q))


def _ladder(sections):
    """each axis has its own ladder of frequencies"""
    return torch.tensor([BASE ** (-i / n) for n in sections for i in range(n)], dtype=torch.float32, device="cuda")


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    if case["op"] == "rope":
        n = case["tokens"]
        sections = _ints(case["sections"])
        # the heads are slices of one projection [tokens, heads + 2 kv_heads, dim], scales differ from channel to channel
        qkv = (normal(n, hq + 2 * hk, d) * torch.exp(0.5 * normal(d))).to(dtype)
        at = torch.arange(n, device="cuda")
        area = case["height"] * case["width"]
        first = int(torch.randint(0, 50000, (1,), generator=g, device="cuda"))       # keyframes are counted from the video's start
        axes = [first + at // area, at % area // case["width"], at % case["width"]]
        s = {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "positions": torch.stack(axes[-len(sections):] if len(sections) > 1 else axes[:1], 1).int(),
             "inv_freq": _ladder(sections), "sections": sections, "q_weight": None, "k_weight": None}
        if case["normalize"]:
            s["q_weight"], s["k_weight"] = 1 + 0.2 * normal(d), 1 + 0.2 * normal(d)
        if case["train"]:
            s["dq"], s["dk"] = normal(n, hq, d).to(dtype), normal(n, hk, d).to(dtype)
        return s
    q_lens, k_lens = _lengths(case)
    nq, nk = sum(q_lens) + case["pad"], sum(k_lens) + case["pad"]
    s = {"q": (1.5 * normal(nq, hq, d)).to(dtype), "k": normal(nk, hk, d).to(dtype), "v": (normal(nk, hk, d) + 0.3 * normal(hk, d)).to(dtype)}
    if case["train"]:
        s["do"] = normal(nq, hq, d).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    grads = {"rope": ("q", "k", "q_weight", "k_weight"), "attn": ("q", "k", "v")}[case["op"]] if case["train"] else ()
    s["leaves"] = [s[n].requires_grad_() if s[n].is_leaf else s[n].detach().requires_grad_() for n in grads if s[n] is not None]
    s.update(zip([n for n in grads if s[n] is not None], s["leaves"]))
    if case["op"] == "attn":
        q_lens, k_lens = _lengths(case)
        if own:
            s["plan"] = _framework().PackedPlan(q_lens, case["heads"], case["kv_heads"], case["dim"], key_lengths=k_lens, causal_block=case["block"], device="cuda")
        else:
            s["q_at"], s["k_at"] = _places(q_lens), _places(k_lens)
    return s


def _places(lens):
    """for sequences of these lengths: length and first row of each, sequence and place of each row, the longest"""
    n = torch.tensor(lens)
    seq = torch.repeat_interleave(torch.arange(len(lens)), n)
    first = torch.cumsum(n, 0) - n
    place = torch.arange(len(seq)) - first[seq]
    return {"n": n.cuda(), "first": first.cuda(), "seq": seq.cuda(), "place": place.cuda(), "most": max(1, max(lens))}


# ----------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        fw = _framework()
        if c["op"] == "rope":
            out = fw.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], s["q_weight"], s["k_weight"], normalize=c["normalize"], eps=EPS,
                                  interleaved=c["interleaved"])
            return tuple(out) + (torch.autograd.grad(out, s["leaves"], (s["dq"], s["dk"])) if c["train"] else ())
        out = fw.packed_attention(s["q"], s["k"], s["v"], s["plan"])
        return (out,) + (torch.autograd.grad(out, s["leaves"], s["do"]) if c["train"] else ())
    with torch.no_grad():
        return _plain_rope(s, c) if c["op"] == "rope" else _plain_attn(s, c)


def _turn(x, cos, sin, pairs, interleaved):
    """rotates the first 2 * pairs channels of x [tokens, heads, dim]"""
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1), x[..., 2 * pairs:]], -1)


def _plain_rope(s, c):
    dtype, sections = s["q"].dtype, s["sections"]
    pairs, mode = sum(sections), c["interleaved"]
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), torch.tensor(sections, device="cuda"), output_size=pairs)
    angle = s["positions"].double()[:, axis] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, dq, wq = _plain_rope_one(s["q"].float(), s["q_weight"], cos, sin, pairs, mode, s["dq"].float() if c["train"] else None, c["normalize"])
    k, dk, wk = _plain_rope_one(s["k"].float(), s["k_weight"], cos, sin, pairs, mode, s["dk"].float() if c["train"] else None, c["normalize"])
    if not c["train"]:
        return q.to(dtype), k.to(dtype)
    return (q.to(dtype), k.to(dtype), dq.to(dtype), dk.to(dtype)) + ((wq, wk) if c["normalize"] else ())


def _plain_rope_one(x, w, cos, sin, pairs, mode, dy, normalize):
    if normalize:
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        y = _turn(x * r * w, cos, sin, pairs, mode)
    else:
        y = _turn(x, cos, sin, pairs, mode)
    if dy is None:
        return y, None, None
    dz = _turn(dy, cos, -sin, pairs, mode)                     # the inverse rotation
    if not normalize:
        return y, dz, None
    dw = (dz * x * r).sum((0, 1), dtype=torch.float64).float()
    dz = dz * w
    return y, r * dz - x * r ** 3 * (dz * x).mean(-1, keepdim=True), dw


def _padded(x, at):
    """packed [rows, heads, dim] -> [sequences, heads, longest, dim] in 32 bits, zero behind the ends"""
    place = torch.arange(at["most"], device="cuda")
    inside = place < at["n"][:, None]
    rows = torch.where(inside, at["first"][:, None] + place, 0)
    return (x[rows].float() * inside[..., None, None]).permute(0, 2, 1, 3).contiguous()


def _packed(x, at, like):
    """[sequences, heads, longest, dim] -> packed, zero in the rows behind the last sequence"""
    rows = x[at["seq"], :, at["place"]]
    return torch.cat([rows, rows.new_zeros(like.shape[0] - rows.shape[0], *rows.shape[1:])]).to(like.dtype)


def _plain_attn(s, c):
    hk, d = c["kv_heads"], c["dim"]
    group, block, scale = c["heads"] // hk, c["block"], 1 / math.sqrt(d)
    qa, ka = s["q_at"], s["k_at"]
    q, k, v = _padded(s["q"], qa), _padded(s["k"], ka), _padded(s["v"], ka)
    n, m, l = len(q), qa["most"], ka["most"]
    q = q.view(n, hk, group * m, d)
    i, j = torch.arange(m, device="cuda"), torch.arange(l, device="cuda")
    end = ka["n"][:, None].expand(n, m)                         # the keys that a query sees are the first `end`
    if block:
        back = i + (ka["n"] - qa["n"])[:, None]                 # the last query stands at the last key
        end = torch.minimum(end, (torch.div(back, block, rounding_mode="floor") + 1) * block)
    hidden = j >= end[:, None, None, :, None]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    p.view(n, hk, group, m, l).masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))                 # a row that sees nothing is zero
    out = _packed(torch.matmul(p, v).view(n, hk * group, m, d), qa, s["q"])
    if not c["train"]:
        return (out,)
    do = _padded(s["do"], qa).view(n, hk, group * m, d)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    dp.sub_((do * torch.matmul(p, v)).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq, dk = torch.matmul(dp, k), torch.matmul(dp.transpose(-1, -2), q)
    return out, _packed(dq.view(n, hk * group, m, d), qa, s["q"]), _packed(dk, ka, s["k"]), _packed(dv, ka, s["v"])


# -------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_rope(s, case) if case["op"] == "rope" else _exact_attn(s, case)


def _exact_rope(s, case):
    """channels as complex numbers, gradients by autograd"""
    names = ["q", "k"] + (["q_weight", "k_weight"] if case["normalize"] else [])
    x = {n: s[n].double().detach().requires_grad_(case["train"]) for n in names}
    sections, pairs = s["sections"], sum(s["sections"])
    parts, at = [], 0
    for a, n in enumerate(sections):
        parts.append(s["positions"][:, a, None].double() * s["inv_freq"][at:at + n].double())
        at += n
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), torch.cat(parts, 1))[:, None]
    out = []
    for n in ("q", "k"):
        z = x[n]
        if case["normalize"]:
            z = z / torch.sqrt((z * z).sum(-1, keepdim=True) / case["dim"] + EPS) * x[n + "_weight"]
        head, rest = z[..., :2 * pairs], z[..., 2 * pairs:]
        if case["interleaved"]:
            y = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (pairs, 2)).contiguous()) * turn).flatten(-2)
        else:
            w = torch.complex(head[..., :pairs], head[..., pairs:]) * turn
            y = torch.cat([w.real, w.imag], -1)
        out.append(torch.cat([y, rest], -1))
    grads = torch.autograd.grad(out, list(x.values()), (s["dq"].double(), s["dk"].double())) if case["train"] else ()
    return tuple(o.detach() for o in out) + tuple(grads)


def _exact_attn(s, case):
    """sequence by sequence, head by head, a slab of queries at a time"""
    q_lens, k_lens = _lengths(case)
    hq, d, block = case["heads"], case["dim"], case["block"]
    group = hq // case["kv_heads"]
    names = ("q", "k", "v") if case["train"] else ()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in names}
    q0 = k0 = 0
    for m, l in zip(q_lens, k_lens):
        slab = max(1, min(m, (1 << 27) // max(1, l)))
        for h in range(hq if m and l else 0):
            k, v = s["k"][k0:k0 + l, h // group].double(), s["v"][k0:k0 + l, h // group].double()
            for a in range(0, m, slab):
                rows = slice(q0 + a, q0 + min(m, a + slab))
                q = s["q"][rows, h].double()
                at = torch.arange(a, a + len(q), device="cuda") + l - m
                sees = torch.full_like(at, l) if not block else (torch.div(at, block, rounding_mode="floor") + 1) * block
                seen = torch.arange(l, device="cuda")[None] < sees[:, None]
                e = torch.where(seen, q @ k.T / math.sqrt(d), -math.inf)
                p = torch.where(seen.any(1, keepdim=True), torch.softmax(e, 1), 0.0)
                o = p @ v
                out[rows, h] = o
                if case["train"]:
                    do = s["do"][rows, h].double()
                    grads["v"][k0:k0 + l, h // group] += p.T @ do
                    de = p * (do @ v.T - (do * o).sum(1, keepdim=True)) / math.sqrt(d)
                    grads["q"][rows, h] = de @ k
                    grads["k"][k0:k0 + l, h // group] += de.T @ q
        q0, k0 = q0 + m, k0 + l
    return (out,) + tuple(grads[n] for n in names)


# ------------------------------------------------------------------------------------------------------------------ the work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        n = case["tokens"]
        values = n * (hq + hk) * d
        small = n * 4 * len(_ints(case["sections"])) + 2 * d * 4 + 4 * sum(_ints(case["sections"]))
        # forward: heads in and out; a training step also takes gradients in and out and reads the heads again
        return {"bytes": (5 if case["train"] else 2) * values * size + small, "flops": values * (30 if case["train"] else 10)}
    q_lens, k_lens = _lengths(case)
    block, pairs = case["block"], 0
    for m, l in zip(q_lens, k_lens):
        pairs += m * l if not block else sum(min(l, max(0, ((i + l - m) // block + 1) * block)) for i in range(m))
    q, kv = sum(q_lens) * hq * d * size, sum(k_lens) * hk * d * size
    # forward: q, k, v in, out written, two products; a training step reads these and the gradient and writes three, five more products
    return {"bytes": 2 * q + 2 * kv + (4 * q + 4 * kv if case["train"] else 0), "flops": (14 if case["train"] else 4) * pairs * hq * d}
