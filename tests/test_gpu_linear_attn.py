"""Linear attention with a decay per head against the recurrence in 64 bits:
lengths around the chunk edges, ragged batches, shared key heads, types,
strides, slots, fresh and padding rows, extreme decays and values."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import layer_oracle as L
from superl8_serve_amd import ops
from tests.kvgpu import DEV, t, to_np

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# What a result may be off, relative to the sum of its terms' absolute values
# (q.k over D dims, tokens and the state's D rows): fp32 sums of at most D + 64
# + D terms and 64 more for the state, 2^-24 each: 448 * 2^-24 < 2^-15.  Where
# a matrix product takes fp32 values as two 16-bit halves, an fp16 pair is
# within 2^-21, a bf16 pair within 2^-16 at worst; three such factors (decayed
# scores, decayed values, the state) on top: fp16 3 * 2^-21 < 2^-19, bf16
# 3 * 2^-16.  Sums: 2^-15 + 2^-19 and 2^-15 + 3 * 2^-16 < 2^-14 * 1.5.
TERMS = {"fp16": 2.0 ** -15 + 2.0 ** -19, "bf16": 2.0 ** -15 + 3 * 2.0 ** -16}


def inputs(rng, n, h, d, dtype, size=1.0):
    return torch.from_numpy((rng.standard_normal((n, h, d)) * size).astype(np.float32)).to(dtype)


def slopes(hq):
    return -np.exp2(-8 * np.arange(1, hq + 1) / hq).astype(np.float32)


def check(what, got, want, room, dtype=None):
    """|got - want| within the terms' room, and half a step of the output's type."""
    got = got.astype(np.float64)
    half = 0.0 if dtype is None else torch.finfo(dtype).eps / 2 * np.abs(want) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    over = np.abs(got - want) - (room + half)
    assert np.isfinite(got).all(), f"{what}: {np.isnan(got).sum()} NaN"
    assert (over <= 0).all(), f"{what}: {over.max():.3e} over at {np.unravel_index(over.argmax(), over.shape)}"


def expect(q, k, v, g, s0, scale, name):
    """(out, state, room of each) of one sequence."""
    f = [x.float().numpy() for x in (q, k, v)]
    out, s = L.linear_attention(*f, g, s0, scale)
    aout, as_ = L.linear_attention(*(np.abs(x) for x in f), g, np.abs(s0), abs(scale))
    return out, s, aout * TERMS[name] + 1e-30, as_ * TERMS[name] + 1e-30


def run(rng, lens, hq, hkv, d, name, g=None, size=1.0, scale=None, slots=None, reset=None, extra_rows=0, views=False):
    dtype = DTYPES[name]
    total, b = sum(lens) + extra_rows, len(lens)
    scale = d ** -0.5 if scale is None else scale
    g = slopes(hq) if g is None else np.asarray(g, np.float32)
    q, k, v = (inputs(rng, total, h, d, dtype, size) for h in (hq, hkv, hkv))
    state = rng.standard_normal((b + 2, hq, d, d)).astype(np.float32) * size * size
    slots = rng.permutation(b + 2)[:b].astype(np.int32) if slots is None else np.asarray(slots, np.int32)
    dev = [x.to(DEV) for x in (q, k, v)]
    if views:  # slices of one projection
        dev = list(torch.cat(dev, 1).split((hq, hkv, hkv), 1))
    pool = t(state)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    out = ops.linear_attn_varlen(*dev, t(g), pool, t(cu), max(lens, default=0), state_slots=t(slots),
                                 reset=None if reset is None else t(np.asarray(reset, bool)), scale=scale)
    got, new = out.float().cpu().numpy(), to_np(pool)
    assert out.dtype == dtype
    left = set(range(b + 2))
    for i in range(b):
        at = slice(cu[i], cu[i + 1])
        if not 0 <= slots[i] < b + 2:
            assert not got[at].any()
            continue
        left.discard(int(slots[i]))
        s0 = state[slots[i]] * (0 if reset is not None and reset[i] else 1)
        wo, ws, ro, rs = expect(q[at], k[at], v[at], g, s0, scale, name)
        check(f"out of sequence {i} ({lens[i]} tokens)", got[at], wo, ro, dtype)
        check(f"state of sequence {i} ({lens[i]} tokens)", new[slots[i]], ws, rs)
    assert not got[cu[-1]:].any()
    for s in left:
        assert np.array_equal(new[s], state[s])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_lengths(d, name):
    rng = np.random.default_rng(d)
    run(rng, [1, 2, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 190], 4, 4, d, name)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_short_sequences(d, name):
    """No more than 32 tokens, whose chunks are half as long; few, which the recurrence takes."""
    rng = np.random.default_rng(d + 1)
    run(rng, [1, 32, 0, 7, 31, 17, 6, 5, 4, 3], 4, 2, d, name, extra_rows=2)
    run(rng, [5, 1, 0, 4], 4, 4, d, name)
    run(rng, [6, 2], 2, 1, d, name, views=True)


@pytest.mark.parametrize("name", list(DTYPES))
def test_short_sequences_in_numbers(name):
    rng = np.random.default_rng(6)
    run(rng, [int(n) for n in rng.integers(0, 140, 70)], 8, 4, 64, name)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_hint_of_32_for_longer_sequences(d, name):
    rng = np.random.default_rng(d + 2)
    q, k, v = (inputs(rng, 200, 2, d, DTYPES[name]) for _ in range(3))
    state = torch.zeros(2, 2, d, d, device=DEV)
    cu = np.array([0, 150, 200], np.int32)
    got = ops.linear_attn_varlen(q.to(DEV), k.to(DEV), v.to(DEV), t(slopes(2)), state, t(cu), 32, scale=0.1).float().cpu().numpy()
    for b in range(2):
        at = slice(cu[b], cu[b + 1])
        wo, ws, ro, rs = expect(q[at], k[at], v[at], slopes(2), np.zeros((2, d, d)), 0.1, name)
        check(f"out {b}", got[at], wo, ro, DTYPES[name])
        check(f"state {b}", to_np(state[b]), ws, rs)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 128), (6, 2, 64), (8, 1, 128), (5, 5, 32), (4, 2, 256)])
def test_heads_views_and_tail(hq, hkv, d, name):
    rng = np.random.default_rng(hq + d)
    run(rng, [70, 5, 200], hq, hkv, d, name, extra_rows=9, views=True)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_long_and_lone(d, name):
    """One sequence on few heads: the tokens are split over workgroups."""
    rng = np.random.default_rng(d + 7)
    run(rng, [3001], 2, 1, d, name)
    run(rng, [1500, 17, 2100], 2, 2, d, name)


@pytest.mark.parametrize("name", list(DTYPES))
def test_slots_and_resets(name):
    rng = np.random.default_rng(12)
    run(rng, [5, 66, 130, 0, 0, 9], 2, 2, 128, name, slots=[3, -1, 0, 7, 8, 6], reset=[True, True, False, True, True, True])
    run(rng, [1, 300], 4, 2, 64, name, slots=[2, 99], reset=[False, False])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_extreme_decays(d, name):
    rng = np.random.default_rng(d)
    run(rng, [150, 64], 8, 8, d, name, g=[0.0, -1e-7, -1e-3, -1.0, -20.0, -90.0, -1e30, -np.inf])
    run(rng, [2500], 2, 2, d, name, g=[0.0, -1e-4])


@pytest.mark.parametrize("size", [1e-3, 60.0, 3000.0])
def test_sizes_of_values(size):
    """Products far outside fp16 in between; the scale brings them back."""
    rng = np.random.default_rng(5)
    run(rng, [200, 33], 2, 2, 128, "fp16", size=size, scale=0.005 / size ** 2)
    run(rng, [200, 33], 2, 2, 128, "bf16", size=size, scale=0.005 / size ** 2)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n", [70, 1000])
def test_nothing_but_the_state(n, name):
    """Values of zero (at first, or all of them) and of the smallest size next to a large state."""
    rng = np.random.default_rng(n)
    d, g = 64, slopes(2)
    q, k, v = (inputs(rng, n, 2, d, DTYPES[name]) for _ in range(3))
    for zero, small in ((64, 1.0), (n, 1.0), (5, 2.0 ** -20)):
        x = v * small
        x[:zero] = 0
        s0 = (rng.standard_normal((2, d, d)) * 2.0 ** 60).astype(np.float32)
        state = t(s0[None])
        cu = t(np.array([0, n], np.int32))
        scale = 2.0 ** -62
        got = ops.linear_attn_varlen(q.to(DEV), k.to(DEV), x.to(DEV), t(g), state, cu, n, scale=scale).float().cpu().numpy()
        wo, ws, ro, rs = expect(q, k, x, g, s0, scale, name)
        check("out", got, wo, ro, DTYPES[name])
        check("state", to_np(state[0]), ws, rs)


def test_unset_max_seqlen_is_only_a_hint():
    rng = np.random.default_rng(3)
    q, k, v = (inputs(rng, 400, 2, 64, torch.float16).to(DEV) for _ in range(3))
    g, cu = t(slopes(2)), t(np.array([0, 390, 400], np.int32))
    state = torch.zeros(2, 2, 64, 64, device=DEV)
    want = ops.linear_attn_varlen(q, k, v, g, state.clone(), cu, 390, scale=0.1)
    for hint in (0, 1, 100, 5000, 100000):
        got = ops.linear_attn_varlen(q, k, v, g, state.clone(), cu, hint, scale=0.1)
        assert (got.float() - want.float()).abs().max() <= 2e-3 * want.float().abs().max()


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("what", ["v", "k", "q", "state"])
def test_non_finite_values_reach_later_tokens_alone(what, name):
    """A NaN or infinity at token 70 leaves the rows before it (of its chunk
    too) and the other heads bit for bit as they are."""
    rng = np.random.default_rng(17)
    q, k, v = (inputs(rng, 200, 2, 128, DTYPES[name]).to(DEV) for _ in range(3))
    g, cu = t(slopes(2)), t(np.array([0, 200], np.int32))
    s0 = torch.randn(1, 2, 128, 128, device=DEV)
    clean = ops.linear_attn_varlen(q, k, v, g, s0.clone(), cu, 200, scale=0.1).float().cpu()
    for bad in (float("nan"), float("inf")):
        x = {"q": q, "k": k, "v": v}
        state = s0.clone()
        if what == "state":
            state[0, 1, 5, 9] = bad
        else:
            x[what] = x[what].clone()
            x[what][70, 1, 9] = bad
        got = ops.linear_attn_varlen(x["q"], x["k"], x["v"], g, state, cu, 200, scale=0.1).float().cpu()
        assert (got[:, 0] - clean[:, 0]).abs().max() <= 2 ** -7 * clean[:, 0].abs().max()
        assert torch.isfinite(got[:, 0]).all()
        if what == "state":
            assert torch.isfinite(got[:, 1, :9]).all() and torch.isfinite(got[:, 1, 10:]).all()
            assert not torch.isfinite(got[:10, 1, 9]).any()
            continue
        assert torch.isfinite(got[:70]).all()
        assert (got[:70] - clean[:70]).abs().max() <= 2 ** -7 * clean[:70].abs().max()
        hit = got[70, 1, 9:10] if what == "v" else got[70, 1]
        assert not torch.isfinite(hit).any()
        if what == "q":
            assert torch.isfinite(got[71:]).all() and torch.isfinite(state).all()
        elif what == "v":
            assert not torch.isfinite(got[71:80, 1, 9]).any()
            assert torch.isfinite(got[70:, 1, :9]).all() and torch.isfinite(got[70:, 1, 10:]).all()


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("b,hq,hkv,d", [(1, 1, 1, 32), (3, 8, 2, 64), (1, 32, 32, 128), (40, 6, 6, 128), (5, 4, 1, 256)])
def test_decode(b, hq, hkv, d, name):
    rng = np.random.default_rng(b + d)
    dtype, scale = DTYPES[name], d ** -0.5
    g = slopes(hq)
    state = rng.standard_normal((b + 2, hq, d, d)).astype(np.float32)
    slots = rng.permutation(b + 2)[:b].astype(np.int32)
    reset = np.zeros(b, bool)
    if b > 2:
        slots[1], reset[2] = -1, True
    pool = t(state)
    for step in range(3):
        q, k, v = (inputs(rng, b, h, d, dtype) for h in (hq, hkv, hkv))
        dev = torch.cat([x.to(DEV) for x in (q, k, v)], 1).split((hq, hkv, hkv), 1)
        out = ops.linear_attn_decode(*dev, t(g), pool, state_slots=t(slots), reset=t(reset), scale=scale)
        got, new = out.float().cpu().numpy(), to_np(pool)
        for i in range(b):
            if slots[i] < 0:
                assert not got[i].any()
                continue
            s0 = state[slots[i]] * (0 if reset[i] else 1)
            wo, ws, ro, rs = expect(q[i:i + 1], k[i:i + 1], v[i:i + 1], g, s0, scale, name)
            check(f"step {step} row {i}", got[i:i + 1], wo, ro, dtype)
            check(f"step {step} state {i}", new[slots[i]], ws, rs)
        for s in set(range(b + 2)) - set(slots.tolist()):
            assert np.array_equal(new[s], state[s])
        state = new


def test_decode_drift():
    """4,000 steps of a slow decay with nothing coming in: the decay's rounding
    does not add up (one fp32 factor alone would be 4000 * 2^-25 off)."""
    d, steps, g = 32, 4000, np.array([-1e-4], np.float32)
    state = torch.ones(1, 1, d, d, device=DEV)
    zero = torch.zeros(1, 1, d, dtype=torch.float16, device=DEV)
    for _ in range(steps):
        ops.linear_attn_decode(zero, zero, zero, t(g) if _ == 0 else dg, state, scale=1.0)
        if _ == 0:
            dg = t(g)
    want = np.exp(np.float64(g[0]) * steps)
    # each step rounds once (random sign): 6 sigma of 4000 roundings of 2^-25 uniform, and the pair's 2^-48
    assert abs(float(state.double().mean()) / want - 1) <= 6 * np.sqrt(steps) * 2.0 ** -25
    assert float((state.double() / want - 1).abs().max()) <= 6 * np.sqrt(steps) * 2.0 ** -25


def test_prompt_in_pieces_equals_whole():
    """A prompt, its chunks, and its tokens one by one leave the same state."""
    rng = np.random.default_rng(23)
    n, hq, d = 150, 3, 64
    q, k, v = (inputs(rng, n, hq, d, torch.float16).to(DEV) for _ in range(3))
    g = t(slopes(hq))
    states = [torch.zeros(1, hq, d, d, device=DEV) for _ in range(3)]
    cu = lambda m: t(np.array([0, m], np.int32))  # noqa: E731
    whole = ops.linear_attn_varlen(q, k, v, g, states[0], cu(n), n, scale=0.125)
    parts = [ops.linear_attn_varlen(q[a:b], k[a:b], v[a:b], g, states[1], cu(b - a), b - a, scale=0.125)
             for a, b in ((0, 40), (40, 104), (104, 150))]
    steps = [ops.linear_attn_decode(q[i:i + 1], k[i:i + 1], v[i:i + 1], g, states[2], scale=0.125) for i in range(n)]
    room = 2 * TERMS["fp16"]
    aout, astate = L.linear_attention(*(np.abs(x.float().cpu().numpy()) for x in (q, k, v)), to_np(g),
                                      np.zeros((hq, d, d)), 0.125)
    for other, state in ((torch.cat(parts), states[1]), (torch.cat(steps), states[2])):
        diff = (other.double() - whole.double()).abs().cpu().numpy()
        assert (diff <= room * aout + 2.0 ** -10 * np.abs(whole.double().cpu().numpy()) + 1e-7).all()
        assert (np.abs(to_np(state).astype(np.float64) - to_np(states[0])) <= room * astate[None]).all()


def test_captured_replays_and_two_streams():
    """Two captured graphs, each with its own workspace, replayed in turn and
    with eager calls between; then two streams at once."""
    rng = np.random.default_rng(41)
    g, cu = t(slopes(2)), t(np.array([0, 700, 2000], np.int32))
    sets = []
    for _ in range(2):
        q, k, v = (inputs(rng, 2000, 2, 64, torch.float16).to(DEV) for _ in range(3))
        state = torch.zeros(2, 2, 64, 64, device=DEV)
        ops.linear_attn_varlen(q, k, v, g, state.clone(), cu, 1300, scale=0.1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_attn_varlen(q, k, v, g, state, cu, 1300, scale=0.1)
            step = ops.linear_attn_decode(q[:2], k[:2], v[:2], g, state, scale=0.1)
        sets.append((q, k, v, state, graph, out, step))
    for i in range(3):
        for q, k, v, state, graph, out, step in sets:
            q.copy_(inputs(rng, 2000, 2, 64, torch.float16))
            eager = state.clone()
            want = ops.linear_attn_varlen(q, k, v, g, eager, cu, 1300, scale=0.1)
            want_step = ops.linear_attn_decode(q[:2], k[:2], v[:2], g, eager, scale=0.1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(step, want_step) and torch.equal(state, eager), f"replay {i}"
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [ops.linear_attn_varlen(*s[:3], g, s[3].clone(), cu, 1300, scale=0.1) for s in sets]
    states = [s[3].clone() for s in sets]
    torch.cuda.synchronize()
    got = []
    for stream, s, state in zip(streams, sets, states):
        with torch.cuda.stream(stream):
            got.append(ops.linear_attn_varlen(*s[:3], g, state, cu, 1300, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_outside_all_sequences():
    rng = np.random.default_rng(51)
    for n in (3, 90):  # the recurrence and the chunks
        q, k, v = (inputs(rng, 2 * n + 20, 2, 64, torch.float16).to(DEV) for _ in range(3))
        cu = np.array([7, 7 + n, 7 + n, 7 + 2 * n], np.int32)
        g, state = t(slopes(2)), torch.zeros(3, 2, 64, 64, device=DEV)
        out = ops.linear_attn_varlen(q, k, v, g, state, t(cu), n, scale=0.1)
        cut = [x[7:7 + 2 * n] for x in (q, k, v)]
        other = torch.zeros_like(state)
        want = ops.linear_attn_varlen(*cut, g, other, t(cu - 7), n, scale=0.1)
        assert not out[:7].any() and not out[7 + 2 * n:].any()
        assert torch.equal(out[7:7 + 2 * n], want) and torch.equal(state, other)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [32, 64, 256])
def test_rows_without_alignment(d, name):
    """Rows that 16-byte loads cannot take."""
    rng = np.random.default_rng(d + 3)
    dtype, lens, hq, hkv = DTYPES[name], [130, 1, 40], 4, 2
    n, cu, g = sum(lens), np.array([0, 130, 131, 171], np.int32), slopes(4)
    wide = [inputs(rng, n, h, d + 2, dtype).to(DEV) for h in (hq, hkv, hkv)]
    q, k, v = (x[:, :, 1:-1] for x in wide)
    state = rng.standard_normal((3, hq, d, d)).astype(np.float32)
    pool = t(state)
    got = ops.linear_attn_varlen(q, k, v, t(g), pool, t(cu), 130, scale=0.1).float().cpu().numpy()
    step = pool.clone()
    one = ops.linear_attn_decode(q[:3], k[:3], v[:3], t(g), step, scale=0.1).float().cpu().numpy()
    q, k, v = (x.cpu() for x in (q, k, v))
    for i in range(3):
        at = slice(cu[i], cu[i + 1])
        wo, ws, ro, rs = expect(q[at], k[at], v[at], g, state[i], 0.1, name)
        check(f"out {i}", got[at], wo, ro, dtype)
        check(f"state {i}", to_np(pool[i]), ws, rs)
        wo, ws, ro, rs = expect(q[i:i + 1], k[i:i + 1], v[i:i + 1], g, to_np(pool[i]), 0.1, name)
        check(f"step {i}", one[i:i + 1], wo, ro, dtype)
        check(f"stepped state {i}", to_np(step[i]), ws, rs)


@pytest.mark.parametrize("hint", [0, 5000])
@pytest.mark.parametrize("what", ["broadcast", "windows"])
def test_rows_that_share_bytes(what, hint):
    """One token's rows for all tokens (stride 0), and rows that overlap the next."""
    rng = np.random.default_rng(13)
    n, hq, d, g = 75, 2, 64, slopes(2)
    if what == "broadcast":
        k, v = (inputs(rng, 1, hq, d, torch.float16).to(DEV).expand(n, hq, d) for _ in range(2))
    else:
        k, v = (inputs(rng, 1, 1, 8 * n + hq * d, torch.float16).to(DEV).as_strided((n, hq, d), (8, d, 1)) for _ in range(2))
    q, state = inputs(rng, n, hq, d, torch.float16), torch.zeros(2, hq, d, d, device=DEV)
    cu = np.array([0, 70, 75], np.int32)
    got = ops.linear_attn_varlen(q.to(DEV), k, v, t(g), state, t(cu), hint, scale=0.1).float().cpu().numpy()
    for b in range(2):
        at = slice(cu[b], cu[b + 1])
        wo, ws, ro, rs = expect(q[at], k.cpu()[at], v.cpu()[at], g, np.zeros((hq, d, d)), 0.1, "fp16")
        check(f"out {b}", got[at], wo, ro, torch.float16)
        check(f"state {b}", to_np(state[b]), ws, rs)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("d", [32, 256])
def test_split_among_short_ones(d, name):
    """Sequences that are split next to short, empty and padding ones."""
    rng = np.random.default_rng(d + 11)
    lens = [30, 0, 1100, 1, 64, 900, 0, 5]
    run(rng, lens, 2, 1, d, name, slots=[4, 5, 0, 9, 1, -1, 2, 3], extra_rows=3)
    run(rng, [700, 65], 2, 2, d, name, reset=[True, False], views=True)


@pytest.mark.parametrize("name", list(DTYPES))
def test_workspace_is_optional(name):
    """The C entry without a workspace, and with one that is too small, runs unsplit."""
    from superl8_serve_amd import _lib

    lib, rng, n, d = _lib.load(), np.random.default_rng(61), 1500, 64
    q, k, v = (inputs(rng, n, 2, d, DTYPES[name]) for _ in range(3))
    dev, g, cu = [x.to(DEV) for x in (q, k, v)], t(slopes(2)), t(np.array([0, n], np.int32))
    need = lib.s8kv_linear_attn_workspace_size(1, 2, d, n, n)
    assert need > 0
    wo, ws, ro, rs = expect(q, k, v, slopes(2), np.zeros((2, d, d)), 0.1, name)
    work = torch.full((need,), 255, dtype=torch.uint8, device=DEV)  # (NaN: what is not written is not read)
    for given, size in ((None, 0), (work, 16), (work, need)):
        state, out = torch.zeros(1, 2, d, d, device=DEV), torch.empty(n, 2, d, dtype=DTYPES[name], device=DEV)
        rc = lib.s8kv_linear_attn_varlen(
            *(a for x in dev for a in (x.data_ptr(), x.stride(0), x.stride(1))), n, 2, 2, d, list(DTYPES).index(name),
            g.data_ptr(), state.data_ptr(), 2 * d * d, 1, None, None, cu.data_ptr(), 1, n, 0.1, out.data_ptr(), 2 * d,
            d, None if given is None else given.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check(f"workspace of {size}", out.float().cpu().numpy(), wo, ro, DTYPES[name])
        check(f"state, workspace of {size}", to_np(state[0]), ws, rs)


@pytest.mark.parametrize("hint", [500, 3000])
@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("what", ["v", "k", "state"])
def test_non_finite_values_stay(what, name, hint):
    """A NaN or infinity early on is in every later output that depends on it,
    across segments and whatever the decay; the other columns (of its wave
    too) stay right over many chunks."""
    rng = np.random.default_rng(71)
    n, d = 3000, 64
    q, k, v = (inputs(rng, n, 2, d, DTYPES[name]) for _ in range(3))
    for g in (np.array([-3.0, -1e-4], np.float32), np.array([-1e-4, 0.0], np.float32)):
        wo, ws, ro, rs = expect(q, k, v, g, np.ones((2, d, d)), 0.1, name)
        keep = np.ones((2, d), bool)
        keep[:, 9] = False
        for bad in (float("nan"), float("inf")):
            x = {"q": q.to(DEV), "k": k.to(DEV), "v": v.to(DEV)}
            state = torch.ones(1, 2, d, d, device=DEV)
            if what == "state":
                state[0, :, 5, 9] = bad
            else:
                x[what][70, :, 9] = bad
            cu = t(np.array([0, n], np.int32))
            got = ops.linear_attn_varlen(x["q"], x["k"], x["v"], t(g), state, cu, hint, scale=0.1).float().cpu().numpy()
            new = to_np(state[0])
            assert not np.isfinite(got[71:, :, 9]).any() and not np.isfinite(new[:, 5 if what == "state" else 9, 9]).any()
            if what == "k":
                assert not np.isfinite(new[:, 9]).any()
                continue
            check("other columns", got[:, keep], wo[:, keep], ro[:, keep], DTYPES[name])
            check("other columns of the state", new.swapaxes(1, 2)[keep], ws.swapaxes(1, 2)[keep], rs.swapaxes(1, 2)[keep])


@pytest.mark.parametrize("name", list(DTYPES))
def test_columns_of_different_sizes(name):
    """Value columns from 2^-12 to 2^6 next to each other, every one to its own size."""
    rng = np.random.default_rng(81)
    n, d = 300, 64
    q, k = (inputs(rng, n, 2, d, DTYPES[name]) for _ in range(2))
    size = np.exp2(np.arange(d) % 19 - 12).astype(np.float32)
    v = torch.from_numpy(rng.uniform(1, 2, (n, 2, d)).astype(np.float32) * size).to(DTYPES[name])
    state = torch.zeros(1, 2, d, d, device=DEV)
    got = ops.linear_attn_varlen(q.to(DEV), k.to(DEV), v.to(DEV), t(slopes(2)), state, t(np.array([0, n], np.int32)), n, scale=0.1)
    wo, ws, ro, rs = expect(q, k, v, slopes(2), np.zeros((2, d, d)), 0.1, name)
    check("out", got.float().cpu().numpy(), wo, ro, DTYPES[name])
    check("state", to_np(state[0]), ws, rs)


def test_slots_past_32_bits():
    """A pool of more than 2^31 elements: slots at its end."""
    hq, d = 32, 256
    slots = 2 ** 31 // (hq * d * d) + 3
    pool = torch.empty(slots, hq, d, d, device=DEV)
    small = torch.randn(2, hq, d, d, device=DEV)
    pool[slots - 2:] = small
    at = t(np.array([slots - 1, slots - 2], np.int32))
    rng = np.random.default_rng(91)
    q, k, v = (inputs(rng, 90, hq, d, torch.bfloat16).to(DEV) for _ in range(3))
    g, cu = t(slopes(hq)), t(np.array([0, 70, 90], np.int32))
    for call in (lambda s, i: ops.linear_attn_varlen(q, k, v, g, s, cu, 70, state_slots=i, scale=0.1),
                 lambda s, i: ops.linear_attn_decode(q[:2], k[:2], v[:2], g, s, state_slots=i, scale=0.1)):
        want = call(small, t(np.array([1, 0], np.int32)))
        assert torch.equal(call(pool, at), want) and torch.equal(pool[slots - 2:], small)


def test_refusals():
    n, hq, hkv, d = 6, 4, 2, 64
    q, k, v = (torch.zeros(n, h, d, dtype=torch.float16, device=DEV) for h in (hq, hkv, hkv))
    g, state = torch.zeros(hq, device=DEV), torch.zeros(3, hq, d, d, device=DEV)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
    ok = dict(q=q, k=k, v=v, log_decay=g, state=state, cu_seqlens=cu, max_seqlen=4, scale=1.0)
    for exc, change in [
        (RuntimeError, dict(q=q.cpu())), (TypeError, dict(q=q.float())), (TypeError, dict(k=k.bfloat16())),
        (ValueError, dict(k=k[:5])), (ValueError, dict(v=v[:, :1])), (ValueError, dict(k=k[:, :0], v=v[:, :0])),
        (ValueError, dict(q=q[:, :3], log_decay=g[:3], state=state[:, :3])),
        (ValueError, dict(log_decay=g[:2])), (TypeError, dict(log_decay=g.double())),
        (TypeError, dict(state=state.half())), (ValueError, dict(state=state.transpose(2, 3))),
        (ValueError, dict(state=state[:, :, :32])), (ValueError, dict(state=state[:1].expand(3, hq, d, d))),
        (TypeError, dict(cu_seqlens=cu.long())), (ValueError, dict(cu_seqlens=cu[:0])), (ValueError, dict(max_seqlen=-1)),
        (ValueError, dict(state_slots=cu)), (TypeError, dict(state_slots=cu[:2].long())),
        (TypeError, dict(reset=cu[:2])), (ValueError, dict(reset=torch.zeros(3, dtype=torch.bool, device=DEV))),
        (RuntimeError, dict(q=torch.zeros(n, 2, 96, dtype=torch.float16, device=DEV),
                            k=torch.zeros(n, 2, 96, dtype=torch.float16, device=DEV),
                            v=torch.zeros(n, 2, 96, dtype=torch.float16, device=DEV), log_decay=g[:2],
                            state=torch.zeros(3, 2, 96, 96, device=DEV))),
    ]:
        with pytest.raises(exc):
            ops.linear_attn_varlen(**{**ok, **change})
    empty = ops.linear_attn_varlen(**{**ok, "cu_seqlens": cu[:1]})
    assert empty.shape == q.shape and not empty.any()
    with pytest.raises(ValueError):
        ops.linear_attn_decode(q, k, v, g, state, state_slots=cu, scale=1.0)
    assert ops.linear_attn_decode(q[:0], k[:0], v[:0], g, state, scale=1.0).shape == (0, hq, d)
