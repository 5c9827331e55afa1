"""The layers of a hybrid model as they run together: prompts through the
rotating cache write, the prefill attention over the fresh rotated keys and the
linear attention; then decode steps of both kinds; then a chunk of drafts
through the verify attention.  Every output against the oracles."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from oracle import layer_oracle as L
from superl8_serve_amd import ops
from superl8_serve_amd.linear_state import LinearStateCache
from superl8_serve_amd.paged_cache import PagedKVCache
from tests.kvgpu import DEV, assert_close, t, to_np
from tests.test_gpu_linear_attn import TERMS, check, slopes

pytestmark = pytest.mark.gpu

HQ, HKV, D, SCALE = 8, 2, 128, 1 / math.sqrt(128)


def rows(rng, n, h, dtype):
    return torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float32)).to(dtype)


def layer_of(c):
    r = [x[0].cpu().numpy() for x in ((c.k_cache, c.k_scale, c.v_packed, c.v_norm, c.v_codebook)
                                      if c.v_quant == "lloydmax3" else (c.k_cache, c.k_scale, c.v_cache, c.v_scale))]
    if c.v_quant == "lloydmax3":
        return O.LayerCache(r[0], r[1], v_packed=r[2], v_norm=r[3], v_codebook=r[4])
    return O.LayerCache(*r)


@pytest.mark.parametrize("v_quant,dtype", [("int8", torch.float16), ("lloydmax3", torch.bfloat16)])
def test_prompts_steps_and_drafts(v_quant, dtype):
    rng = np.random.default_rng(77)
    lens, steps, drafts = [70, 1, 133], 3, 4
    paged = PagedKVCache(1, 4, HKV, 512, D, device=DEV, block_size=16, v_quant=v_quant)
    slots = [paged.alloc() for _ in lens]
    paged.ensure_capacity(slots, [n + steps + drafts for n in lens])
    linear = LinearStateCache(1, 5, HQ, D, device=DEV)
    linear.state.fill_(float("nan"))  # what a slot's last user left is not read
    at = [linear.alloc() for _ in lens]
    table, g = L.cos_sin_table(512, D, 1e6), slopes(HQ)
    wq, wk = (1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32)
    norms = dict(q_norm=t(wq), k_norm=t(wk))
    name = "fp16" if dtype == torch.float16 else "bf16"
    hist = [[] for _ in lens]  # q, k, v of the linear layer, all tokens so far

    def oracle_rope(x, pos, w):
        return torch.from_numpy(L.rope(x.float().numpy(), pos, table, norm=w)).half()

    def linear_check(what, out, per_seq):
        got, first = out.float().cpu().numpy(), 0
        for b, new in enumerate(per_seq):
            hist[b].append(new)
            q, k, v = (torch.cat([h[i] for h in hist[b]]).float().numpy() for i in range(3))
            n = new[0].shape[0]
            want, s = L.linear_attention(q, k, v, g, np.zeros((HQ, D, D)), SCALE)
            room, s_room = L.linear_attention(np.abs(q), np.abs(k), np.abs(v), g, np.zeros((HQ, D, D)), SCALE)
            calls = len(hist[b])  # (each call rounds the state it carries on once more)
            check(f"{what} {b}", got[first:first + n], want[-n:], calls * TERMS[name] * room[-n:] + 1e-30, dtype)
            check(f"{what} state {b}", to_np(linear.state[0, at[b]]), s, calls * TERMS[name] * s_room + 1e-30)
            first += n

    # ---- prompts ----
    total, pos = sum(lens), np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    q, k, v = (rows(rng, total, h, dtype) for h in (HQ, HKV, HKV))
    mapping = torch.cat([torch.tensor(paged.flat_slot_mapping(s, n), dtype=torch.int32) for s, n in zip(slots, lens)]).to(DEV)
    fused = torch.cat([q, k, v], 1).to(DEV).split((HQ, HKV, HKV), 1)  # one projection's views
    fresh = torch.empty(total, HKV, D, dtype=torch.float16, device=DEV)
    rq = paged.write_varlen_rope(0, mapping, *fused, t(pos), t(table), k_out=fresh, **norms)
    cu = t(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    out = ops.attn_varlen(rq, fresh, v.half().to(DEV), cu, cu, max(lens), max(lens), causal=True, scale=SCALE)
    want_q, want_k = oracle_rope(q, pos, wq), oracle_rope(k, pos, wk)
    assert torch.equal(rq.cpu(), want_q) and torch.equal(fresh.cpu(), want_k)
    first = 0
    for n in lens:
        s = slice(first, first + n)
        qq, kk, vv = want_q[s].double(), want_k[s].double().repeat_interleave(HQ // HKV, 1), v[s].half().double().repeat_interleave(HQ // HKV, 1)
        p = torch.einsum("ihd,jhd->hij", qq, kk) * SCALE
        p = p.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf).softmax(-1)
        assert_close(out[s].float().cpu().numpy(), torch.einsum("hij,jhd->ihd", p, vv).numpy(), f"prefill of {n}")
        first += n
    lq, lk, lv = (rows(rng, total, h, dtype) for h in (HQ, HKV, HKV))
    lout = linear.attn_varlen(0, lq.to(DEV), lk.to(DEV), lv.to(DEV), t(g), at, lens, scale=SCALE)
    linear_check("prompt", lout, list(zip(lq.split(lens), lk.split(lens), lv.split(lens))))

    # ---- decode steps ----
    ctx = list(lens)
    for step in range(steps):
        b = len(lens)
        q, k, v = (rows(rng, b, h, dtype) for h in (HQ, HKV, HKV))
        rq = paged.write_decode_rope(0, slots, ctx, q.to(DEV), k.to(DEV), v.to(DEV), t(table), **norms)
        out = paged.decode_attn(0, rq.unsqueeze(2), slots, ctx, scale=SCALE)
        assert torch.equal(rq.cpu(), oracle_rope(q, np.array(ctx), wq))
        bt = paged.block_table(slots).cpu().numpy()
        ctx = [n + 1 for n in ctx]
        want = O.paged_decode(to_np(rq), layer_of(paged), bt, np.array(ctx), SCALE)
        assert_close(out[:, :, 0].float().cpu().numpy(), want, f"decode step {step}")
        lq, lk, lv = (rows(rng, b, h, dtype) for h in (HQ, HKV, HKV))
        lout = linear.attn_decode(0, lq.to(DEV), lk.to(DEV), lv.to(DEV), t(g), at, scale=SCALE)
        linear_check(f"step {step}", lout, list(zip(lq.split(1), lk.split(1), lv.split(1))))

    # ---- a chunk of drafts behind each sequence ----
    b = len(lens)
    q, k, v = (rows(rng, b * drafts, h, dtype) for h in (HQ, HKV, HKV))
    pos = np.concatenate([np.arange(n, n + drafts) for n in ctx]).astype(np.int32)
    mapping = paged.slot_mapping_for([s for s in slots for _ in range(drafts)], pos.tolist())
    rq = paged.write_varlen_rope(0, mapping, q.to(DEV), k.to(DEV), v.to(DEV), t(pos), t(table), **norms)
    out = paged.verify_attn(0, rq.reshape(b, drafts, HQ, D).transpose(1, 2), slots, ctx, scale=SCALE)
    bt, rot = paged.block_table(slots).cpu().numpy(), to_np(rq).reshape(b, drafts, HQ, D)
    for i in range(drafts):
        want = O.paged_decode(rot[:, i], layer_of(paged), bt, np.array(ctx) + i + 1, SCALE)
        assert_close(out[:, :, i].float().cpu().numpy(), want, f"draft {i}")


def test_state_cache_slots():
    c = LinearStateCache(2, 3, 1, 32, device=DEV)
    a, b = c.alloc(), c.alloc()
    assert (a, b) == (2, 1) and c.has_free_slot()
    g = torch.zeros(1, device=DEV)
    x = torch.ones(2, 1, 32, dtype=torch.float16, device=DEV)
    c.attn_decode(0, x, x, x, g, [a, b], scale=1.0)
    c.attn_decode(0, x, x, x, g, [a, b], scale=1.0)
    assert (c.state[0, [a, b]] == 2).all() and not c.state[0, 0].any() and not c.state[1].any()
    c.free(a)
    assert c.alloc() == a
    with pytest.raises(ValueError):
        c.attn_decode(0, x[:1], x, x, g, [a], scale=1.0)
    c.attn_decode(0, x[:1], x[:1], x[:1], g, [a], scale=1.0)  # fresh again in layer 0, a refused call later too
    c.attn_varlen(1, x, x, x, g, [b], [2], scale=1.0)
    assert (c.state[0, a] == 1).all() and (c.state[0, b] == 2).all() and (c.state[1, b] == 2).all()
    for bad in (lambda: c.attn_decode(0, x, x, x, g, [a, a], scale=1.0), lambda: c.attn_decode(0, x, x, x, g, [a, 3], scale=1.0),
                lambda: c.attn_varlen(0, x, x, x, g, [a], [1], scale=1.0), lambda: c.free(0), lambda: c.free(7),
                lambda: c.attn_varlen(0, x, x, x, g, [a, b], [3, -1], scale=1.0)):
        with pytest.raises(ValueError):
            bad()
    c.alloc()
    assert not c.has_free_slot()
    with pytest.raises(RuntimeError):
        c.alloc()
