"""Rotary positions (``ops.rope``) and the rotating cache writes, bit for bit
against the oracle: types, head layouts, pairings, partial heads, several
position axes, norms, strides and alignments, tokens without a slot."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from oracle import layer_oracle as L
from superl8_serve_amd import ops
from tests.kvgpu import CODEBOOK, DEV, alloc, t, to_np

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def rows(rng, n, h, d, dtype, outliers=True):
    x = rng.standard_normal((n, h, d)).astype(np.float32)
    if outliers:
        x[..., rng.integers(0, d)] *= 20
    return torch.from_numpy(x).to(dtype)


def positions(rng, n, axes, top):
    p = rng.integers(0, top, (axes, n)).astype(np.int32)
    return p if axes > 1 else p[0]


def want_rope(x, pos, table, dtype, **how):
    """The oracle's rows in the output's type (torch rounds to the nearest even)."""
    with np.errstate(over="ignore"):
        return torch.from_numpy(L.rope(x.float().numpy(), pos, table, **how)).to(dtype)


def same(got, want):
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = (got != want) & ~nan
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values differ, first at {bad.nonzero()[0].tolist()}"


CASES = [
    # d, rot, hq, hkv, pairing, sections, interleaved, norm, tokens
    (128, 128, 32, 8, "half", None, False, True, 65),
    (128, 128, 16, 8, "half", None, False, False, 1),
    (128, 64, 7, 1, "half", None, False, True, 19),
    (128, 32, 3, 3, "half", None, False, False, 8),
    (128, 16, 5, 2, "half", None, False, True, 9),
    (128, 96, 4, 2, "half", None, False, True, 9),
    (128, 126, 4, 2, "adjacent", None, False, True, 5),
    (128, 112, 8, 2, "adjacent", None, False, False, 33),
    (128, 128, 28, 4, "half", (16, 24, 24), False, False, 70),
    (128, 128, 8, 4, "half", (24, 20, 20), True, True, 35),
    (128, 64, 8, 4, "adjacent", (8, 8, 8, 8), False, True, 35),
    (256, 256, 16, 4, "half", None, False, True, 21),
    (256, 64, 16, 4, "adjacent", None, False, False, 130),
    (256, 256, 4, 2, "adjacent", (64, 64), True, True, 17),
    (256, 256, 4, 1, "half", (100, 20, 8), False, False, 6),
    (64, 64, 32, 8, "half", None, False, True, 77),
    (64, 32, 9, 3, "half", (8, 4, 4), True, False, 12),
    (64, 16, 2, 2, "half", None, False, True, 40),
    (32, 32, 12, 4, "half", None, False, True, 51),
    (32, 16, 4, 1, "half", (4, 4), False, True, 50),
    (32, 8, 4, 1, "adjacent", None, False, False, 3),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d,rot,hq,hkv,pairing,sections,interleaved,norm,n", CASES)
def test_rope_bits(d, rot, hq, hkv, pairing, sections, interleaved, norm, n, dtype):
    rng = np.random.default_rng(d + rot + hq + n)
    table = L.cos_sin_table(300, rot)
    pos = positions(rng, n, len(sections) if sections else 1, 300)
    q, k = rows(rng, n, hq, d, DTYPES[dtype]), rows(rng, n, hkv, d, DTYPES[dtype])
    how = dict(sections=sections, interleaved=interleaved, pairing=pairing)
    wq, wk = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32) if norm else (None, None)
    gq, gk = ops.rope(q.to(DEV), k.to(DEV), t(pos), t(table), q_norm=None if wq is None else t(wq),
                      k_norm=None if wk is None else t(wk), eps=1e-5, **how)
    same(gq, want_rope(q, pos, table, q.dtype, norm=wq, eps=1e-5, **how))
    same(gk, want_rope(k, pos, table, k.dtype, norm=wk, eps=1e-5, **how))


@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("wdtype", ["fp16", "bf16", "fp32"])
def test_rope_views_in_place_and_alone(shift, wdtype):
    """q and k as slices of one projection (any alignment), rotated in place,
    and q without k; norm weights in each type."""
    rng = np.random.default_rng(3 + shift)
    d, n = 128, 23
    table, pos = L.cos_sin_table(100, d), positions(rng, n, 1, 100)
    w = torch.from_numpy((1 + 0.3 * rng.standard_normal(d)).astype(np.float32)).to(DTYPES[wdtype])
    fused = torch.zeros(n, 12 * d + shift, dtype=torch.float16, device=DEV)
    host = rows(rng, n, 12, d, torch.float16)
    fused[:, shift:] = host.reshape(n, -1).to(DEV)
    q, k, rest = fused[:, shift:].reshape(n, 12, d).split((8, 2, 2), 1) if shift == 0 else \
        fused[:, shift:].unflatten(1, (12, d)).split((8, 2, 2), 1)
    wn = w.float().numpy()
    want_q, want_k = (want_rope(x, pos, table, torch.float16, norm=wn) for x in (host[:, :8], host[:, 8:10]))
    alone, none = ops.rope(q, None, t(pos), t(table), q_norm=w.to(DEV))
    assert none is None
    same(alone, want_q)
    got_q, got_k = ops.rope(q, k, t(pos), t(table), q_norm=w.to(DEV), k_norm=w.to(DEV), q_out=q, k_out=k)
    assert got_q is q and got_k is k
    same(got_q, want_q)
    same(got_k, want_k)
    same(rest, host[:, 10:])  # the other rows of the projection are left as they were
    if shift:
        assert not fused[:, :shift].any()


def test_rope_positions_outside_the_table_and_no_tokens():
    rng = np.random.default_rng(9)
    table = L.cos_sin_table(50, 64)
    pos = np.array([0, -1, 49, 50, 2**31 - 1, -2**31], np.int32)
    q = rows(rng, 6, 4, 128, torch.bfloat16)
    got, _ = ops.rope(q.to(DEV), None, t(pos), t(table))
    same(got, want_rope(q, pos, table, torch.bfloat16))
    assert torch.isnan(got[1, :, :64]).all() and torch.isfinite(got[1, :, 64:]).all()
    empty, _ = ops.rope(q[:0].to(DEV), None, t(pos[:0]), t(table))
    assert empty.shape == (0, 4, 128)


def oracle_write(kind, k, v, slots, n_blocks, bs):
    hkv, d = k.shape[1:]
    cache = [to_np(x) for x in alloc(kind, n_blocks, hkv, bs, d)]
    with np.errstate(invalid="ignore", over="ignore"):
        if kind == "int8":
            O.quantize_kv_write_paged(k, v, *cache, slots)
        else:
            O.k8v3_write_paged(k, v, *cache, CODEBOOK, slots)
    return cache


def write(kind, q, k, v, pos, table, cache, slots, **how):
    if kind == "int8":
        return ops.quantize_kv_write_paged_rope(q, k, v, pos, table, *cache, slots, **how)
    return ops.quantize_kv_write_paged_k8v3_rope(q, k, v, pos, table, *cache, t(CODEBOOK), slots, **how)


def same_cache(cache, want):
    for name, g, w in zip(("k", "k scale", "v", "v scale / norm"), cache, want):
        g = to_np(g)
        assert np.array_equal(g.view(np.uint8), w.view(np.uint8)), f"{name}: {(g != w).sum()} of {g.size} values differ"


# (K8V3 has head_dim 128 and 256)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind,d,rot,hq,hkv,pairing,sections,interleaved,norm,n",
                         [(kind, *c) for kind in ("int8", "k8v3") for c in CASES if kind == "int8" or c[0] >= 128])
def test_write_bits(kind, d, rot, hq, hkv, pairing, sections, interleaved, norm, n, dtype):
    rng = np.random.default_rng(d + rot + hq + n + 1)
    bs, n_blocks = 16, n // 16 + 9
    table = L.cos_sin_table(300, rot)
    pos = positions(rng, n, len(sections) if sections else 1, 300)
    q, k, v = (rows(rng, n, h, d, DTYPES[dtype]) for h in (hq, hkv, hkv))
    v[n // 2] = 0  # a zero row: scale 0
    slots = rng.permutation(n_blocks * bs)[:n].astype(np.int32)
    if n > 4:
        slots[1], slots[3] = -1, n_blocks * bs + 5  # neither writes
    how = dict(sections=sections, interleaved=interleaved, pairing=pairing)
    wq, wk = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32) if norm else (None, None)
    cache = alloc(kind, n_blocks, hkv, bs, d)
    k_out = torch.empty(n, hkv, d, dtype=torch.float16, device=DEV)
    gq = write(kind, q.to(DEV), k.to(DEV), v.to(DEV), t(pos), t(table), cache, t(slots), k_out=k_out,
               q_norm=None if wq is None else t(wq), k_norm=None if wk is None else t(wk), **how)
    want_k = want_rope(k, pos, table, torch.float16, norm=wk, **how)
    same(gq, want_rope(q, pos, table, torch.float16, norm=wq, **how))
    same(k_out, want_k)
    keep = (slots >= 0) & (slots < n_blocks * bs)
    same_cache(cache, oracle_write(kind, want_k.numpy()[keep], v.half().numpy()[keep], slots[keep], n_blocks, bs))


@pytest.mark.parametrize("kind", ["int8", "k8v3"])
def test_write_equals_rope_then_append(kind):
    """The one launch against the two calls it replaces, 2,000 tokens of one
    projection's views with three axes."""
    rng = np.random.default_rng(21)
    n, hq, hkv, d, bs = 2000, 28, 4, 128, 64
    heads = rows(rng, n, hq + 2 * hkv, d, torch.float16).to(DEV)
    q, k, v = heads.split((hq, hkv, hkv), 1)
    pos, table = t(positions(rng, n, 3, 4000)), t(L.cos_sin_table(4000, d, 1e6))
    slots = t(rng.permutation(40 * bs)[:n].astype(np.int32))
    how = dict(sections=(16, 24, 24), q_norm=torch.full((d,), 1.5, device=DEV), k_norm=torch.full((d,), 0.7, device=DEV))
    one, two = alloc(kind, 40, hkv, bs, d), alloc(kind, 40, hkv, bs, d)
    gq = write(kind, q, k, v, pos, table, one, slots, **how)
    rq, rk = ops.rope(q, k, pos, table, **how)
    if kind == "int8":
        ops.quantize_kv_write_paged(rk, v, *two, slots)
    else:
        ops.quantize_kv_write_paged_k8v3(rk, v, *two, t(CODEBOOK), slots)
    same(gq, rq)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["int8", "k8v3"])
def test_write_past_32_bits(kind):
    """A cache of more than 2^32 bytes: the rows at its end are the append's."""
    hkv, d, bs = 8, 128, 16
    blocks = 2 ** 32 // (hkv * d * bs) + 4
    rng = np.random.default_rng(99)
    q, k, v = (torch.from_numpy(rng.standard_normal((3, h, d)).astype(np.float16)).to(DEV) for h in (16, hkv, hkv))
    pos, table = t(np.array([0, 5, 70], np.int32)), t(L.cos_sin_table(128, d))
    cb = t(np.sort(rng.standard_normal(8)).astype(np.float32))

    def cache(n):
        e = lambda dtype, *last: torch.empty(n, hkv, bs, *last, dtype=dtype, device=DEV)  # noqa: E731
        if kind == "int8":
            return [e(torch.int8, d), e(torch.float32), e(torch.int8, d), e(torch.float32)]
        return [e(torch.int8, d), e(torch.float32), e(torch.int32, 12), e(torch.float32, 1), cb]

    small, large = cache(4), cache(blocks)
    at = np.array([63, 0, 17], np.int32)
    rq, rk = ops.rope(q, k, pos, table)
    if kind == "int8":
        ops.quantize_kv_write_paged(rk, v, *small, t(at))
        got = ops.quantize_kv_write_paged_rope(q, k, v, pos, table, *large, t(at + (blocks - 4) * bs))
    else:
        ops.quantize_kv_write_paged_k8v3(rk, v, *small, t(at), 128)
        got = ops.quantize_kv_write_paged_k8v3_rope(q, k, v, pos, table, *large, t(at + (blocks - 4) * bs), 128)
    assert torch.equal(got, rq)
    for a, b in zip(small[:4], large[:4]):
        for s in at:
            assert torch.equal(a[s // bs, :, s % bs], b[blocks - 4 + s // bs, :, s % bs])


@pytest.mark.parametrize("kind", ["int8", "k8v3"])
@pytest.mark.parametrize("shift", [0, 3])
def test_write_non_finite_rows_stay_apart(kind, shift):
    """Infinities and NaN in one token's rows reach that token's outputs alone
    (the cache bytes are the append's for such rows)."""
    rng = np.random.default_rng(4)
    n, hq, hkv, d, bs = 24, 4, 2, 128, 16
    host = [rows(rng, n, h, d, torch.float16) for h in (hq, hkv, hkv)]
    host[0][3, 1, 5] = float("nan")
    host[1][7, 0, 9], host[1][8, 1, 64] = float("inf"), float("nan")
    host[2][9, 1, 100], host[2][10, 0, 1] = float("-inf"), float("nan")
    dev = []
    for x in host:
        f = torch.zeros(n, x.shape[1] * d + shift, dtype=torch.float16, device=DEV)[:, shift:].unflatten(1, (x.shape[1], d))
        f.copy_(x)
        dev.append(f)
    pos, table = positions(rng, n, 1, 60), L.cos_sin_table(60, d)
    slots = rng.permutation(4 * bs)[:n].astype(np.int32)
    one, two = alloc(kind, 4, hkv, bs, d), alloc(kind, 4, hkv, bs, d)
    k_out = torch.empty(n, hkv, d, dtype=torch.float16, device=DEV)
    gq = write(kind, *dev, t(pos), t(table), one, t(slots), k_out=k_out)
    want_k = want_rope(host[1], pos, table, torch.float16)
    same(gq, want_rope(host[0], pos, table, torch.float16))
    same(k_out, want_k)
    if kind == "int8":
        ops.quantize_kv_write_paged(k_out, dev[2], *two, t(slots))
    else:
        ops.quantize_kv_write_paged_k8v3(k_out, dev[2], *two, t(CODEBOOK), t(slots))
    for a, b in zip(one, two):
        assert np.array_equal(to_np(a).view(np.uint8), to_np(b).view(np.uint8))


def test_write_captured_replays_with_new_inputs_and_streams():
    rng = np.random.default_rng(31)
    n, hq, hkv, d, bs = 40, 8, 2, 128, 16
    table = t(L.cos_sin_table(600, d))
    q, k, v = (rows(rng, n, h, d, torch.float16).to(DEV) for h in (hq, hkv, hkv))
    pos, slots = t(positions(rng, n, 1, 600)), t(rng.permutation(8 * bs)[:n].astype(np.int32))
    cache, q_out = alloc("int8", 8, hkv, bs, d), torch.empty(n, hq, d, dtype=torch.float16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        write("int8", q, k, v, pos, table, cache, slots, q_out=q_out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write("int8", q, k, v, pos, table, cache, slots, q_out=q_out)
    for i in range(3):
        for x in (q, k, v):
            x.copy_(rows(rng, n, x.shape[1], d, torch.float16))
        pos.copy_(t(positions(rng, n, 1, 600)))
        slots.copy_(t(rng.permutation(8 * bs)[:n].astype(np.int32)))
        want = [x.clone() for x in cache]
        want_q = write("int8", q, k, v, pos, table, want, slots)
        graph.replay()
        torch.cuda.synchronize()
        same(q_out, want_q)
        for a, b in zip(cache, want):
            assert torch.equal(a, b), f"replay {i}"


def test_write_large_pool_offsets():
    """Rows past 4 GiB of a layer's K tensor."""
    rng = np.random.default_rng(8)
    hkv, bs, d = 8, 256, 128
    n_blocks = (1 << 32) // (hkv * bs * d) + 3
    cache = [torch.empty((n_blocks, hkv, bs, d), dtype=torch.int8, device=DEV),
             torch.empty((n_blocks, hkv, bs), device=DEV),
             torch.empty((n_blocks, hkv, bs, d), dtype=torch.int8, device=DEV),
             torch.empty((n_blocks, hkv, bs), device=DEV)]
    slots = np.array([0, n_blocks * bs - 1, (n_blocks - 2) * bs + 7], np.int32)
    q, k, v = (rows(rng, 3, h, d, torch.float16) for h in (8, hkv, hkv))
    pos, table = positions(rng, 3, 1, 60), L.cos_sin_table(60, d)
    ops.quantize_kv_write_paged_rope(q.to(DEV), k.to(DEV), v.to(DEV), t(pos), t(table), *cache, t(slots))
    kw, ks = O.quantize_i8_rowwise(O.rotate_last(want_rope(k, pos, table, torch.float16).numpy()))
    vw, vs = O.quantize_i8_rowwise(v.numpy())
    for i, s in enumerate(slots):
        at = (int(s) // bs, slice(None), int(s) % bs)
        for got, want in zip(cache, (kw[i], ks[i], vw[i], vs[i])):
            assert np.array_equal(to_np(got[at]), want)


def test_refusals():
    rng = np.random.default_rng(0)
    n, hq, hkv, d, bs = 6, 4, 2, 128, 16
    q, k, v = (rows(rng, n, h, d, torch.float16).to(DEV) for h in (hq, hkv, hkv))
    pos, table = torch.zeros(n, dtype=torch.int32, device=DEV), t(L.cos_sin_table(20, d))
    slots, cache = torch.zeros(n, dtype=torch.int32, device=DEV), alloc("int8", 2, hkv, bs, d)
    for exc, args, how in [
        (RuntimeError, (q.cpu(), k, pos, table), {}),
        (TypeError, (q, k.float(), pos, table), {}),
        (TypeError, (q.double(), None, pos, table), {}),
        (TypeError, (q, k, pos.long(), table), {}),
        (TypeError, (q, k, pos, table.half()), {}),
        (ValueError, (q, k[:5], pos, table), {}),
        (ValueError, (q, k[..., :64], pos, table), {}),
        (ValueError, (q, k, pos[:5], table), {}),
        (ValueError, (q, k, pos, t(L.cos_sin_table(20, 256))), {}),
        (ValueError, (q, k, pos, table[:, :127]), {}),
        (ValueError, (q, k, pos, table[:0]), {}),
        (ValueError, (q, k, pos, table), {"pairing": "both"}),
        (ValueError, (q, k, pos, table), {"interleaved": True}),
        (ValueError, (q, k, pos, table), {"sections": (32, 32)}),
        (ValueError, (q, k, pos.expand(2, n), table), {"sections": (32, 31)}),
        (ValueError, (q, k, pos.expand(5, n), table), {"sections": (20, 20, 20, 2, 2)}),
        (ValueError, (q, k, pos.expand(2, n), table), {"sections": (24, 40), "interleaved": True}),
        (ValueError, (q, k, pos, table), {"q_norm": torch.ones(64, device=DEV)}),
        (ValueError, (q, k, pos, table), {"q_norm": torch.ones(d, device=DEV), "k_norm": torch.ones(d, device=DEV).half()}),
        (TypeError, (q, k, pos, table), {"q_out": torch.empty_like(q).float()}),
        (ValueError, (q, k, pos, table), {"q_out": torch.empty_like(q)[:5]}),
        (ValueError, (q, None, pos, table), {"k_out": k}),
        (RuntimeError, (torch.zeros(n, 2, 96, dtype=torch.float16, device=DEV), None, pos, t(L.cos_sin_table(20, 96))), {}),
    ]:
        with pytest.raises(exc):
            ops.rope(*args, **how)
    for exc, args in [
        (TypeError, (q.float(), k.float(), v.float(), pos, table, *cache, slots)),
        (ValueError, (q, k, v[:, :1], pos, table, *cache, slots)),
        (ValueError, (q, k, v, pos, table, *cache, slots[:3])),
        (TypeError, (q, k, v, pos, table, *cache, slots.long())),
        (ValueError, (q, k, v, pos, table, cache[0], cache[1], cache[2][:1], cache[3], slots)),
        (TypeError, (q, k, v, pos, table, cache[0].float(), *cache[1:], slots)),
    ]:
        with pytest.raises(exc):
            ops.quantize_kv_write_paged_rope(*args)
    k8 = alloc("k8v3", 2, hkv, bs, d)
    with pytest.raises(RuntimeError):
        ops.quantize_kv_write_paged_k8v3_rope(q, k, v, pos, table, *k8, t(CODEBOOK), slots, 64)
