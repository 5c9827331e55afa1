"""Host-side refusals of the ops of rotary positions and linear attention that
need no GPU: host tensors, and the C entry points' own checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from superl8_serve_amd import _lib, ops


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    pos, table = torch.zeros(2, dtype=torch.int32), torch.zeros(8, 64)
    kc, ks = torch.zeros(2, 4, 16, 64, dtype=torch.int8), torch.ones(2, 4, 16)
    state, g, cu = torch.zeros(1, 4, 64, 64), torch.zeros(4), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.rope(q, q, pos, table),
                 lambda: ops.quantize_kv_write_paged_rope(q, q, q, pos, table, kc, ks, kc, ks, pos),
                 lambda: ops.quantize_kv_write_paged_k8v3_rope(q, q, q, pos, table, kc, ks, pos, ks, g, pos),
                 lambda: ops.linear_attn_varlen(q, q, q, g, state, cu, 2, scale=1.0),
                 lambda: ops.linear_attn_decode(q, q, q, g, state, scale=1.0)):
        with pytest.raises(RuntimeError):
            call()


def test_axis_maps():
    amap = list(ops._axis_map((2, 3, 3), False, 8))
    assert [amap[0] >> 2 * p & 3 for p in range(8)] == [0, 0, 1, 1, 1, 2, 2, 2] and amap[1:] == [0, 0, 0]
    amap = list(ops._axis_map((24, 20, 20), True, 64))
    axes = [amap[p // 32] >> 2 * (p % 32) & 3 for p in range(64)]
    assert axes[:6] == [0, 1, 2, 0, 1, 2] and axes[58:] == [1, 2, 0, 0, 0, 0] and [axes.count(a) for a in (0, 1, 2)] == [24, 20, 20]
    for bad in ((8,), (2, 3, 4), (-1, 9), (2, 2, 2, 1, 1)):
        with pytest.raises(ValueError):
            ops._axis_map(bad, False, 8)
    with pytest.raises(ValueError):
        ops._axis_map((3, 5), True, 8)  # five interleaved pairs of axis 1 need nine


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libsuperl8_kv.so not built")
def test_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p = 4096  # never read: every call is refused before a launch
    ok = dict(q=p, hq=4, qt=256, qh=64, k=p, hk=2, kt=128, kh=64, t=3, d=64, dtype=0, pos=p, axes=1, stride=0, amap=None,
              table=p, rows=10, rot=64, pairing=0, qn=None, kn=None, nd=0, eps=1e-6, qo=p, qot=256, qoh=64, ko=p, kot=128,
              koh=64, stream=None)
    for change, rc, word in [({"d": 96}, -2, b"head_dim"), ({"hq": 0}, -1, b"heads"), ({"t": -1}, -1, b"tokens"),
                             ({"rot": 63}, -1, b"rot_dim"), ({"rot": 66}, -1, b"rot_dim"), ({"pairing": 2}, -1, b"pairing"),
                             ({"axes": 5}, -1, b"axes"), ({"axes": 2}, -1, b"axes"), ({"rows": 0}, -1, b"table"),
                             ({"pos": None}, -1, b"null"), ({"q": None}, -1, b"null"), ({"ko": None}, -1, b"null"),
                             ({"dtype": 3}, -1, b"dtype"),
                             ({"axes": 2, "amap": (ctypes.c_uint64 * 4)(2, 0, 0, 0)}, -1, b"axis")]:
        assert lib.s8kv_rope(*{**ok, **change}.values()) == rc, change
        assert word in lib.s8kv_last_error(), (change, lib.s8kv_last_error())
    assert lib.s8kv_rope(*{**ok, "t": 0}.values()) == 0
    cache = dict(slots=p, kc=p, ks=p, vc=p, vs=p, blocks=4, bs=16, stream=None)
    head = {**{x: ok[x] for x in ("q", "hq", "qt", "qh", "k")}, "v": p, **{x: ok[x] for x in ("hk", "kt", "kh")},
            "vt": 128, "vh": 64, **{x: ok[x] for x in list(ok)[8:-1]}}
    for change, rc, word in [({"dtype": 2}, -1, b"dtype"), ({"bs": 12}, -2, b"block_size"), ({"blocks": 0}, -1, b"num_blocks"),
                             ({"v": None}, -1, b"null"), ({"slots": None}, -1, b"null"), ({"ks": None}, -1, b"null"),
                             ({"hk": 0}, -1, b"kv"), ({"blocks": 1 << 40}, -2, b"2^32")]:
        assert lib.s8kv_append_rope_int8(*{**head, **cache, **change}.values()) == rc, change
        assert word in lib.s8kv_last_error(), (change, lib.s8kv_last_error())
    lin = dict(q=p, qt=128, qh=64, k=p, kt=64, kh=64, v=p, vt=64, vh=64, t=5, hq=2, hk=1, d=64, dtype=0, g=p, state=p,
               slot=8192, slots=3, at=None, reset=None, cu=p, b=2, longest=4, scale=1.0, out=p, ot=128, oh=64, ws=None, wsb=0,
               stream=None)
    for change, rc, word in [({"d": 48}, -2, b"head_dim"), ({"dtype": 2}, -1, b"dtype"), ({"hk": 0}, -1, b"kv"),
                             ({"hq": 3, "hk": 2}, -1, b"multiple"), ({"slot": 8191}, -1, b"slots"), ({"state": None}, -1, b"state"),
                             ({"state": 4100}, -1, b"aligned"), ({"cu": None}, -1, b"null"), ({"g": None}, -1, b"null"),
                             ({"longest": -1}, -1, b"max_seqlen"), ({"t": 1 << 31}, -1, b"32 bits"), ({"b": -1}, -1, b"sequences")]:
        assert lib.s8kv_linear_attn_varlen(*{**lin, **change}.values()) == rc, change
        assert word in lib.s8kv_last_error(), (change, lib.s8kv_last_error())
    assert lib.s8kv_linear_attn_varlen(*{**lin, "b": 0}.values()) == 0
    assert lib.s8kv_linear_attn_workspace_size(0, 2, 64, 100, 100) == 0
    assert lib.s8kv_linear_attn_workspace_size(1, 2, 64, 100000, 100000) > 0


def test_devices_other_than_the_current_one_become_current(monkeypatch):
    """A launch goes to the tensors' device (here without a GPU: the switch is recorded)."""
    seen = []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            seen.append(self.device.index)

        def __exit__(self, *e):
            seen.append("back")

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    assert ops._launch(torch.device("cuda:0"), lambda *a: a, 1, 2) == (1, 2) and seen == []
    assert ops._launch(torch.device("cuda:1"), lambda *a: a, 3) == (3,) and seen == [1, "back"]
