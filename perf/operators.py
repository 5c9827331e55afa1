"""Performance cases of what a layer does around the paged KV cache: rotary
positions, the cache write with the rotation on the way, and linear attention
with a decay per head (the other layers of a hybrid model).

A case is a dict of plain values.  ``prepare`` makes what the engine holds
before the call, ``run`` is one pass: the plain form in elementary torch
operations, or (``own``) the framework's op; ``exact`` the same outputs from
the definition in 64 bits; ``work`` the bytes and operations that the pass
cannot do without.

Kinds of pass:
  rope     q and k of ``tokens`` tokens rotated by their positions (``axes`` 3:
           time, height and width, as images have them)
  write    the same on the way into a paged cache: q out, k and v quantized;
           the cache's contents come back as the values they stand for
  linear   causal linear attention of a ragged batch of prompts (or a few
           drafts each), states read from and left in a pool
  step     its form for one token a sequence

Sizes that a case does not spell out (lengths, slots, positions) come from its
``shape_seed``; values come from the seed given to ``prepare``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
#: Lloyd-Max levels of N(0, 1) at 8 levels (Max 1960), the 3-bit V codebook before its 1/sqrt(128).
LEVELS = (0.2451, 0.7560, 1.3439, 2.1520)
BLOCK = 128
CHUNK = 256  # tokens a step of the plain linear attention


def _ops():
    from superl8_serve_amd import ops

    return ops


def _rope(name, **kw):
    return {"name": name, "kind": "rope", "dtype": "float16", "d": 128, "rot": 128, "pairing": "half", "axes": 1,
            "interleaved": False, "norm": False, **kw}


def _write(name, **kw):
    return {**_rope(name, **kw), "kind": "write", "layout": "int8", "bs": 256, **kw}


def listed():
    return [
        # one user's decode step, the small model's heads: latency is all there is
        _rope("rope_1", tokens=1, hq=16, hkv=8, norm=True, shape_seed=1),
        # an image and text prompt: time, height and width positions
        _rope("rope_image_prompt", tokens=7001, hq=32, hkv=8, dtype="bfloat16", axes=3, interleaved=True, shape_seed=2),
        # a batch of prompts on a model that rotates a quarter of its 256-wide heads, adjacent pairs
        _rope("rope_partial_d256", tokens=12289, hq=16, hkv=4, d=256, rot=64, pairing="adjacent", shape_seed=3),
        # the ordinary decode step of one layer: 64 users, normalised heads
        _write("write_64", tokens=64, hq=32, hkv=8, norm=True, bs=16, shape_seed=4),
        # one chunk of prompts of the same model
        _write("write_16k", tokens=16384, hq=32, hkv=8, norm=True, shape_seed=5),
        # an image prompt into the 3-bit V layout, odd sizes, few KV heads, small blocks
        _write("write_k8v3", tokens=4099, hq=28, hkv=4, axes=3, dtype="bfloat16", layout="k8v3", bs=16, shape_seed=6),
        # a lone long document
        {"name": "linear_1_long", "kind": "linear", "dtype": "float16", "batch": 1, "hq": 32, "hkv": 32, "d": 128,
         "lo": 32768, "hi": 32768, "shape_seed": 7},
        # a ragged batch of prompts
        {"name": "linear_ragged", "kind": "linear", "dtype": "bfloat16", "batch": 12, "hq": 32, "hkv": 32, "d": 128,
         "lo": 200, "hi": 4000, "shape_seed": 8},
        # a few drafts for each of many users, shared key heads of 64
        {"name": "linear_drafts", "kind": "linear", "dtype": "float16", "batch": 32, "hq": 32, "hkv": 8, "d": 64,
         "lo": 5, "hi": 5, "shape_seed": 9},
        # one user's next token
        {"name": "step_1", "kind": "step", "dtype": "bfloat16", "batch": 1, "hq": 32, "hkv": 32, "d": 128, "shape_seed": 10},
        # the ordinary decode step: 64 users
        {"name": "step_64", "kind": "step", "dtype": "float16", "batch": 64, "hq": 32, "hkv": 32, "d": 128,
         "shape_seed": 11},
    ]


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 1.0e9 and w["flops"] <= 6.8e10:  # no dearer than the listed long document
            return case


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw(rng):
    kind = rng.choice(("rope", "write", "write", "linear", "linear", "step"))
    d = rng.choice((128, 128, 128, 64, 256))
    hkv = rng.choice((1, 2, 4, 8, 8))
    case = {"kind": kind, "dtype": rng.choice(("float16", "bfloat16")), "d": d, "hkv": hkv,
            "hq": hkv * rng.choice((1, 2, 4, 5, 7, 8)), "shape_seed": rng.randrange(1 << 30)}
    if kind in ("rope", "write"):
        rot = d // rng.choice((1, 1, 1, 2, 4))
        axes = rng.choice((1, 1, 3)) if rot >= 32 else 1
        case |= {"tokens": _log(rng, 1, 16384), "rot": rot, "pairing": rng.choice(("half", "half", "adjacent")),
                 "axes": axes, "interleaved": axes > 1 and rng.random() < 0.5, "norm": rng.random() < 0.5}
        if kind == "write":
            layout = rng.choice(("int8", "int8", "k8v3")) if d >= 128 else "int8"
            case |= {"layout": layout, "bs": rng.choice((16, 64, 256)) if case["tokens"] > 256 else 16}
        return case
    case |= {"batch": _log(rng, 1, 64), "d": rng.choice((64, 128, 128)), "hkv": 8 * rng.choice((1, 2, 4))}
    case["hq"] = case["hkv"] * rng.choice((1, 1, 2))
    if kind == "linear":
        hi = _log(rng, 1, 16384)
        case |= {"hi": hi, "lo": max(1, hi // rng.choice((1, 2, 4, 16)))}
    return case


# ---------------------------------------------------------------------------
# Sizes of a case
# ---------------------------------------------------------------------------


def _lens(case):
    r = random.Random(case["shape_seed"])
    if case["kind"] == "step":
        return [1] * case["batch"]
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _sections(case):
    """Pairs of each axis: a half for time, a quarter each for height and width (about)."""
    if case["axes"] == 1:
        return None
    half = case["rot"] // 2
    side = half // 4 if case["interleaved"] else half * 3 // 8
    return (half - 2 * side, side, side)


def _axis_of_pair(case):
    half, sections = case["rot"] // 2, _sections(case)
    if sections is None:
        return [0] * half
    if not case["interleaved"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [p % 3 if p < 3 * sections[p % 3] else 0 for p in range(half)]


def _cell(case):
    """Cache bytes of one token and KV head: int8 K and its scale, and V."""
    d = case["d"]
    return d + 4 + (d + 4 if case["layout"] == "int8" else 3 * d // 8 + 4 * (d // BLOCK))


def work(case):
    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    if case["kind"] in ("rope", "write"):
        t = case["tokens"]
        place = t * (4 * case["axes"] + 4 * case["rot"])  # positions, and a table row
        flops = t * (hq + hkv) * (3 * case["rot"] + (3 * d if case["norm"] else 0))
        if case["kind"] == "rope":
            return {"bytes": place + 4 * t * (hq + hkv) * d, "flops": flops}
        fwht = int(d * math.log2(d))
        return {"bytes": place + t * (4 * hq * d + hkv * (4 * d + _cell(case)) + 4),
                "flops": flops + t * hkv * (fwht + 6 * d)}
    tokens, states = sum(_lens(case)), 8 * case["batch"] * hq * d * d
    return {"bytes": states + 4 * tokens * (hq + hkv) * d, "flops": 4 * d * d * hq * tokens}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _table(rows, rot):
    """cos | sin of every position, from angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = torch.arange(rows, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _positions(case):
    """[axes, tokens]: prompts behind each other; with three axes an image's rows and columns between text."""
    r, t = random.Random(case["shape_seed"]), case["tokens"]
    first = r.randint(0, 20000)
    if case["kind"] == "write" and t <= 256:  # a decode step: every token deep in a sequence of its own
        time = [r.randint(0, 30000) for _ in range(t)]
    else:
        time = [first + i % 5000 for i in range(t)]
    if case["axes"] == 1:
        return [time]
    wide = r.randint(8, 60)
    image = [i % 1500 >= 400 for i in range(t)]
    grid = [(i % 1500 - 400) for i in range(t)]
    return [[x - g if im else x for x, g, im in zip(time, grid, image)],
            [x - g + g // wide if im else x for x, g, im in zip(time, grid, image)],
            [x - g + g % wide if im else x for x, g, im in zip(time, grid, image)]]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    d, hq, hkv, dtype = case["d"], case["hq"], case["hkv"], getattr(torch, case["dtype"])
    st = {"case": case}
    if case["kind"] in ("rope", "write"):
        t = case["tokens"]
        # one projection's output, split: q, k and v are views of it
        heads = _randn(gen, t, hq + 2 * hkv, d)
        heads[..., torch.randperm(d, generator=gen, device=DEV)[: d // 64]] *= 20  # outlier channels
        st["q"], st["k"], st["v"] = heads.to(dtype).split((hq, hkv, hkv), 1)
        at = _positions(case)
        st["positions"] = _int32(at) if case["axes"] > 1 else _int32(at[0])
        st["table"] = _table(32768, case["rot"])
        st["axis"] = torch.tensor(_axis_of_pair(case), device=DEV)
        st["how"] = {"pairing": case["pairing"], "sections": _sections(case), "interleaved": case["interleaved"]}
        if case["norm"]:
            st["how"] |= {"q_norm": 1 + 0.2 * _randn(gen, d), "k_norm": 1 + 0.2 * _randn(gen, d), "eps": EPS}
        if case["kind"] == "write":
            bs = case["bs"]
            per = bs if t > 256 else 1  # decode rows: a block each
            blocks = -(-t // per) + 2
            order = random.Random(case["shape_seed"]).sample(range(blocks), blocks)
            r = random.Random(case["shape_seed"] + 1)
            off = [i % bs if per == bs else r.randrange(bs) for i in range(t)]
            st["slots"] = _int32([order[i // per] * bs + off[i] for i in range(t)])
            head = (blocks, hkv, bs)
            st["pool"] = {"k_cache": torch.zeros((*head, d), dtype=torch.int8, device=DEV),
                          "k_scale": torch.ones(head, device=DEV)}
            if case["layout"] == "int8":
                st["pool"] |= {"v_cache": torch.zeros((*head, d), dtype=torch.int8, device=DEV),
                               "v_scale": torch.ones(head, device=DEV)}
            else:
                st["pool"] |= {"v_packed": torch.zeros((*head, 3 * d // 32), dtype=torch.int32, device=DEV),
                               "v_norm": torch.ones((*head, d // BLOCK), device=DEV)}
            levels = [-v for v in reversed(LEVELS)] + list(LEVELS)
            st["codebook"] = torch.tensor(levels, device=DEV) / math.sqrt(BLOCK)
        return st
    lens = _lens(case)
    total, ends = sum(lens), [0]
    for n in lens:
        ends.append(ends[-1] + n)
    # queries and keys behind an activation, as such layers have them
    st["q"] = torch.nn.functional.silu(_randn(gen, total, hq, d)).to(dtype)
    st["k"] = torch.nn.functional.silu(_randn(gen, total, hkv, d)).to(dtype)
    st["v"] = _randn(gen, total, hkv, d).to(dtype)
    st["decay"] = -torch.exp2(-8 * torch.arange(1, hq + 1, device=DEV) / hq)
    slots = random.Random(case["shape_seed"]).sample(range(case["batch"] + 3), case["batch"])
    st["slots"] = _int32(slots)
    st["state"] = _randn(gen, case["batch"] + 3, hq, d, d)
    st["cu"], st["longest"], st["scale"] = _int32(ends), max(lens), d ** -0.5
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _angles(st):
    """cos and sin [T, 1, R/2] of each pair at its axis's position."""
    half = st["table"].shape[1] // 2
    at = st["positions"].reshape(-1, st["q"].shape[0])[st["axis"]].long()  # [R/2, T]
    pair = torch.arange(half, device=DEV).unsqueeze(1)
    return st["table"][at, pair].T.unsqueeze(1), st["table"][at, pair + half].T.unsqueeze(1)


def _rotated(st, x, weight):
    """x in 32 bits, normalised (where the model does) and rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    c, s = st["angles"]
    rot = st["table"].shape[1]
    if st["how"]["pairing"] == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., rot:]], -1)


def _hadamard(d, dtype):
    """The normalised Sylvester matrix: the sign is the parity of the common bits of row and column."""
    i = torch.arange(d, device=DEV)
    common = i.unsqueeze(1) & i
    bits = common ^ common >> 4
    bits = bits ^ bits >> 2
    return (1 - 2 * ((bits ^ bits >> 1) & 1)).to(dtype) / math.sqrt(d)


def _codes(y):
    """Symmetric int8 codes of each row, and its scale."""
    scale = (y.abs().amax(-1) / torch.full((), 127, dtype=y.dtype, device=DEV)).float()
    by = scale.to(y.dtype).clamp_min(1e-30).unsqueeze(-1)
    return (y / by).round().clamp(-127, 127).to(torch.int8), scale


def _lloyd(v, codebook):
    """3-bit codes of each row's 128-value blocks (nearest level) and the blocks' norms."""
    blocks = v.reshape(*v.shape[:-1], -1, BLOCK)
    norm = blocks.square().sum(-1).sqrt()
    edges = ((codebook[1:] + codebook[:-1]) / 2).to(v.dtype)
    return torch.bucketize(blocks / norm.clamp_min(1e-30).unsqueeze(-1), edges).reshape(v.shape), norm.float()


def _pack(codes):
    """Bit-plane words: word 3 g + b holds bit b of codes 32 g .. 32 g + 31."""
    c = codes.reshape(*codes.shape[:-1], -1, 1, 32)
    bit = torch.arange(3, device=DEV).reshape(3, 1)
    words = ((c >> bit & 1) << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int().flatten(-2)


def _unpack(words):
    w = words.reshape(*words.shape[:-1], -1, 3, 1)
    bits = w >> torch.arange(32, device=DEV, dtype=torch.int32) & 1
    return (bits[..., 0, :] + 2 * bits[..., 1, :] + 4 * bits[..., 2, :]).flatten(-2)


def _values(st):
    """What the pool stands for (K as stored, rotated), in fp16 as its readers have it."""
    pool = st["pool"]
    k = pool["k_cache"] * pool["k_scale"].half().unsqueeze(-1)
    if "v_cache" in pool:
        return k, pool["v_cache"] * pool["v_scale"].half().unsqueeze(-1)
    codes = _ops().unpack_codes3(pool["v_packed"], k.shape[-1]).int() if own else _unpack(pool["v_packed"])
    v = torch.nn.functional.embedding(codes, st["codebook"].half().unsqueeze(-1)).reshape(*k.shape[:-1], -1, BLOCK)
    return k, (v * pool["v_norm"].half().unsqueeze(-1)).reshape(k.shape)


def _run_write(st):
    how, pool = st["how"], st["pool"]
    if own:
        cache = [t for t in pool.values()] + ([st["codebook"]] if "v_packed" in pool else [])
        op = _ops().quantize_kv_write_paged_k8v3_rope if "v_packed" in pool else _ops().quantize_kv_write_paged_rope
        q = op(st["q"], st["k"], st["v"], st["positions"], st["table"], *cache, st["slots"], **how)
    else:
        st["angles"] = _angles(st)
        q = _rotated(st, st["q"], how.get("q_norm")).half()
        k = _rotated(st, st["k"], how.get("k_norm")).half().float()
        bs = pool["k_cache"].shape[2]
        blk, off = st["slots"].long() // bs, st["slots"].long() % bs
        y = (k @ _hadamard(k.shape[-1], k.dtype)).half().float()
        pool["k_cache"][blk, :, off], pool["k_scale"][blk, :, off] = _codes(y)
        v = st["v"].half().float()
        if "v_cache" in pool:
            pool["v_cache"][blk, :, off], pool["v_scale"][blk, :, off] = _codes(v)
        else:
            codes, pool["v_norm"][blk, :, off] = _lloyd(v, st["codebook"])
            pool["v_packed"][blk, :, off] = _pack(codes)
    k, v = _values(st)
    return {"q": q, "k": k, "v": v}


def _linear(q, k, v, decay, state, scale):
    """One sequence, [n, H, D] in 32 bits: outputs, and the state after it."""
    outs = []
    for at in range(0, q.shape[0], CHUNK):
        qc, kc, vc = (x[at: at + CHUNK].transpose(0, 1) for x in (q, k, v))  # [H, n, D]
        n = qc.shape[1]
        i = torch.arange(n, device=DEV)
        ago = (i.unsqueeze(1) - i).float()
        mask = torch.exp(decay.reshape(-1, 1, 1) * ago.clamp_min(0)) * (ago >= 0)
        since = torch.exp(decay.unsqueeze(1) * (i + 1)).unsqueeze(-1)
        left = torch.exp(decay.unsqueeze(1) * (n - 1 - i)).unsqueeze(-1)
        outs.append((qc @ kc.transpose(1, 2) * mask) @ vc + qc * since @ state)
        state = state * torch.exp(decay * n).reshape(-1, 1, 1) + (kc * left).transpose(1, 2) @ vc
    return torch.cat(outs, 1).transpose(0, 1) * scale, state


def _run_linear(st):
    case, state = st["case"], st["state"]
    if own:
        how = {"state_slots": st["slots"], "scale": st["scale"]}
        if case["kind"] == "step":
            out = _ops().linear_attn_decode(st["q"], st["k"], st["v"], st["decay"], state, **how)
        else:
            out = _ops().linear_attn_varlen(st["q"], st["k"], st["v"], st["decay"], state, st["cu"], st["longest"], **how)
        return {"out": out, "state": state}
    group, slots = case["hq"] // case["hkv"], st["slots"].long()
    q, k, v = st["q"].float(), (st["k"].float().repeat_interleave(group, 1)), (st["v"].float().repeat_interleave(group, 1))
    if case["kind"] == "step":
        new = state[slots] * torch.exp(st["decay"]).reshape(-1, 1, 1) + k.unsqueeze(-1) * v.unsqueeze(-2)
        out = (q.unsqueeze(-2) @ new).squeeze(-2) * st["scale"]
        state[slots] = new
        return {"out": out.to(st["q"].dtype), "state": state}
    outs, news, lens = [], [], _lens(case)
    for b, (x, y, z) in enumerate(zip(q.split(lens), k.split(lens), v.split(lens))):
        out, new = _linear(x, y, z, st["decay"], state[slots[b]], st["scale"])
        outs.append(out)
        news.append(new)
    state[slots] = torch.stack(news)
    return {"out": torch.cat(outs).to(st["q"].dtype), "state": state}


def run(st):
    kind = st["case"]["kind"]
    if kind == "write":
        return _run_write(st)
    if kind != "rope":
        return _run_linear(st)
    if own:
        q, k = _ops().rope(st["q"], st["k"], st["positions"], st["table"], **st["how"])
        return {"q": q, "k": k}
    st["angles"] = _angles(st)
    dtype = st["q"].dtype
    return {"q": _rotated(st, st["q"], st["how"].get("q_norm")).to(dtype),
            "k": _rotated(st, st["k"], st["how"].get("k_norm")).to(dtype)}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_rotated(st, x, weight):
    """Each pair as a complex number times its unit complex number."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    half = st["table"].shape[1] // 2
    at = st["positions"].reshape(-1, x.shape[0])
    unit = torch.empty((x.shape[0], half), dtype=torch.complex128, device=DEV)
    for p, a in enumerate(_axis_of_pair(st["case"])):
        rows = st["table"][at[a].long()].double()
        unit[:, p] = torch.complex(rows[:, p], rows[:, half + p])
    out = x.clone()
    first = slice(0, half) if st["how"]["pairing"] == "half" else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if st["how"]["pairing"] == "half" else slice(1, 2 * half, 2)
    turned = torch.complex(x[..., first], x[..., second]) * unit.unsqueeze(1)
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _exact_write(st):
    """The stored values follow the cache's definition: K rounded to fp16 as a layer hands it over, the
    Hadamard product rounded to fp16, codes to the nearest."""
    pool, how = st["pool"], st["how"]
    d, bs = pool["k_cache"].shape[-1], pool["k_cache"].shape[2]
    h = torch.ones((1, 1), dtype=torch.float64, device=DEV)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    k = _exact_rotated(st, st["k"], how.get("k_norm")).half().double()
    y = (k @ h / math.sqrt(d)).half().double()

    def steps(x):
        scale = x.abs().amax(-1, keepdim=True) / 127
        return torch.where(scale > 0, (x / scale).round() * scale, 0)

    v = st["v"].half().double()
    if "v_cache" in pool:
        v = steps(v)
    else:
        blocks = v.reshape(*v.shape[:-1], -1, BLOCK)
        norm = blocks.pow(2).sum(-1, keepdim=True).sqrt()
        levels = st["codebook"].double()
        near = (blocks / norm).unsqueeze(-1).sub(levels).abs().argmin(-1)
        v = (levels[near] * norm).reshape(v.shape)
    kk = torch.zeros(pool["k_cache"].shape, dtype=torch.float64, device=DEV)
    # rows that nothing wrote stand for zeros (int8) or for the first level times a norm of one
    vv = torch.zeros_like(kk) if "v_cache" in pool else torch.full_like(kk, float(st["codebook"][0]))
    blk, off = st["slots"].long() // bs, st["slots"].long() % bs
    kk[blk, :, off], vv[blk, :, off] = steps(y), v
    return {"q": _exact_rotated(st, st["q"], how.get("q_norm")), "k": kk, "v": vv}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "write":
        return _exact_write(st)
    if case["kind"] == "rope":
        return {"q": _exact_rotated(st, st["q"], st["how"].get("q_norm")),
                "k": _exact_rotated(st, st["k"], st["how"].get("k_norm"))}
    # the recurrence, token by token, all sequences and heads at once
    lens, slots, group = _lens(case), st["slots"].long(), case["hq"] // case["hkv"]
    n = torch.tensor(lens, device=DEV)
    first = st["cu"][:-1].long()
    lam = st["decay"].double().exp().reshape(-1, 1, 1)
    s = st["state"][slots].double()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for t in range(max(lens)):
        live = torch.tensor([b for b, m in enumerate(lens) if t < m], device=DEV) if min(lens) <= t else slice(None)
        at = first[live] + t
        k, v = (st[x][at].double().repeat_interleave(group, 1) for x in ("k", "v"))
        new = torch.addcmul(s[live] * lam, k.unsqueeze(-1), v.unsqueeze(-2))
        s[live] = new
        out[at] = (st["q"][at].double().unsqueeze(-2) @ new).squeeze(-2) * st["scale"]
    state = st["state"].double()
    state[slots] = s
    return {"out": out, "state": state}
