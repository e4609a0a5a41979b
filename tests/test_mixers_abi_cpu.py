"""CPU checks of the token mixers' C entry points and bindings: refusals before any CUDA call, workspace sizes,
struct layouts. No kernel is launched here."""
from __future__ import annotations

import ctypes
import struct

import pytest
import torch

A16 = 0x10000  # aligned, never dereferenced: validation fails first
A8 = 0x10008


def cache(wz, **kw):
    c = wz.KvCache(A16, A16, A16, A16, None, None, None, None, 1024, 4096)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn_args(wz, c, **kw):
    a = wz.KvAttnArgs()
    d = dict(q=A16, q_heads=16, q_head_stride=256, q_row_stride=4096, out=A16, out_head_stride=256, out_row_stride=4096,
             lse=None, source=wz.KV_RING, kv_heads=2, head_dim=256, d_base_pos=None, pos_offset=0, window=128, sinks=4,
             scale=0.0625, workspace=A16, workspace_bytes=1 << 40)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    a.cache = ctypes.pointer(c) if c is not None else None
    return a


@pytest.mark.parametrize("fn", ["wzyb_kv_attn_f16", "wzyb_kv_attn_f32"])
def test_attn_refusals(wz, fn):
    f = getattr(wz.lib(), fn)

    def rc(T=4, c=None, **kw):
        return f(ctypes.byref(attn_args(wz, c or cache(wz), **kw)), T, None)

    assert f(None, 4, None) == wz.ERR_NULL
    assert f(ctypes.byref(attn_args(wz, None)), 4, None) == wz.ERR_NULL
    assert rc(q=None) == wz.ERR_NULL and rc(out=None) == wz.ERR_NULL
    assert rc(c=cache(wz, ring_v_s=None)) == wz.ERR_NULL
    assert rc(source=wz.KV_FULL) == wz.ERR_NULL  # no mirror given
    assert rc(workspace=None) == wz.ERR_NULL
    assert rc(source=2) == wz.ERR_VALUE
    assert rc(T=-1) == wz.ERR_SHAPE and rc(T=(1 << 22) + 1) == wz.ERR_SHAPE
    assert rc(kv_heads=0) == wz.ERR_SHAPE and rc(kv_heads=65, q_heads=65) == wz.ERR_SHAPE
    assert rc(kv_heads=3) == wz.ERR_SHAPE  # 16 query heads
    assert rc(q_heads=0) == wz.ERR_SHAPE and rc(q_heads=258) == wz.ERR_SHAPE
    assert rc(head_dim=96) == wz.ERR_SHAPE
    assert rc(window=-1) == wz.ERR_SHAPE and rc(sinks=-1) == wz.ERR_SHAPE
    assert rc(c=cache(wz, ring_cap=0)) == wz.ERR_SHAPE and rc(c=cache(wz, max_ctx=1 << 31)) == wz.ERR_SHAPE
    assert rc(out_head_stride=128) == wz.ERR_SHAPE  # heads of out would overlap
    assert rc(out_row_stride=2048) == wz.ERR_SHAPE
    assert rc(q_row_stride=-4096) == wz.ERR_SHAPE
    assert rc(workspace_bytes=wz.kv_attn_workspace_bytes(4, 16, 2, 256) - 1) == wz.ERR_SHAPE
    for name in ("q", "out", "workspace"):
        assert rc(**{name: A8}) == wz.ERR_ALIGN
    assert rc(q_head_stride=257) == wz.ERR_ALIGN and rc(q_row_stride=4097) == wz.ERR_ALIGN
    assert rc(lse=A16 + 2) == wz.ERR_ALIGN
    for name in ("ring_k_q", "ring_k_s", "ring_v_q", "ring_v_s"):
        assert rc(c=cache(wz, **{name: A8})) == wz.ERR_ALIGN
    assert rc(T=0) == wz.OK


@pytest.mark.parametrize("fn", ["wzyb_kv_tree_attn_f16", "wzyb_kv_tree_attn_f32"])
def test_tree_refusals(wz, fn):
    f = getattr(wz.lib(), fn)
    c, d = cache(wz), cache(wz, ring_cap=40)
    a = attn_args(wz, c)

    def rc(n=40, drafts=d, mask=A16, depth=A16):
        return f(ctypes.byref(a), ctypes.byref(drafts) if drafts is not None else None, mask, depth, n, None)

    assert rc(drafts=None) == wz.ERR_NULL and rc(mask=None) == wz.ERR_NULL and rc(depth=None) == wz.ERR_NULL
    assert rc(drafts=cache(wz, ring_k_q=None)) == wz.ERR_NULL
    assert rc(n=41) == wz.ERR_SHAPE  # more nodes than draft cells
    assert rc(n=wz.TREE_MAX_NODES + 1, drafts=cache(wz, ring_cap=4096)) == wz.ERR_SHAPE
    assert rc(drafts=cache(wz, ring_v_q=A8)) == wz.ERR_ALIGN
    assert rc(mask=A16 + 2) == wz.ERR_ALIGN and rc(depth=A16 + 1) == wz.ERR_ALIGN
    assert rc(n=0) == wz.OK


@pytest.mark.parametrize("fn", ["wzyb_gdn_delta_rule_f16", "wzyb_gdn_delta_rule_f32"])
def test_gdn_refusals(wz, fn):
    f = getattr(wz.lib(), fn)

    def rc(T=4, **kw):
        a = wz.GdnDeltaArgs()
        d = dict(q=A16, k=A16, v=A16, q_row_stride=2048, k_row_stride=2048, v_row_stride=4096, g=A16, beta=A16, state_in=A16,
                 state_out=A16, state_snaps=None, o=A16, o_row_stride=4096, k_heads=16, v_heads=32, head_dim=128, scale=0.1,
                 qk_l2norm=1, l2_eps=1e-6, workspace=A16, workspace_bytes=1 << 40)
        d.update(kw)
        for k, v in d.items():
            setattr(a, k, v)
        return f(ctypes.byref(a), T, None)

    assert f(None, 4, None) == wz.ERR_NULL
    for name in ("q", "k", "v", "g", "beta", "o", "state_out"):
        assert rc(**{name: None}) == wz.ERR_NULL
    assert rc(T=-1) == wz.ERR_SHAPE
    assert rc(head_dim=256) == wz.ERR_SHAPE and rc(head_dim=96) == wz.ERR_SHAPE
    assert rc(k_heads=0) == wz.ERR_SHAPE and rc(k_heads=15) == wz.ERR_SHAPE and rc(v_heads=1040) == wz.ERR_SHAPE
    assert rc(q_row_stride=1024) == wz.ERR_SHAPE and rc(o_row_stride=4095) == wz.ERR_SHAPE
    for name in ("q", "k", "v", "o", "state_in", "state_out", "state_snaps"):
        assert rc(**{name: A8}) == wz.ERR_ALIGN
    assert rc(g=A16 + 2) == wz.ERR_ALIGN
    assert rc(v_row_stride=4097) == wz.ERR_ALIGN
    assert rc(T=0) == wz.OK  # state_in is state_out: nothing to do


def test_workspace_sizes(wz):
    assert wz.kv_attn_workspace_bytes(0, 16, 2, 256) == 0
    assert wz.kv_attn_workspace_bytes(4096, 16, 2, 256) == 0  # enough row tiles without splitting the keys
    assert 0 < wz.kv_attn_workspace_bytes(1, 16, 2, 256) < 1 << 24
    for T in (1, 2, 3, 8, 26, 64, 200, 1021):
        assert wz.kv_attn_workspace_bytes(T, 24, 2, 256) < 1 << 28
    assert wz.gdn_delta_rule_workspace_bytes(1, 16, 32) >= 0


def test_packed_structs_match(wz):
    """The one-call packing of the argument structs has the ctypes (and so the C) layout."""
    vals = list(range(1, 20))
    vals[16] = 0.5
    raw = wz._KV_ATTN_PACK(*vals)
    assert len(raw) == ctypes.sizeof(wz.KvAttnArgs)
    a = wz.KvAttnArgs.from_buffer_copy(raw)
    for (name, _), v in zip(wz.KvAttnArgs._fields_, vals):
        got = getattr(a, name)
        assert (ctypes.cast(got, ctypes.c_void_p).value if name == "cache" else got) == v, name
    vals = list(range(1, 22))
    vals[16], vals[18] = 0.5, 0.25
    raw = wz._GDN_DELTA_PACK(*vals)
    assert len(raw) == ctypes.sizeof(wz.GdnDeltaArgs)
    a = wz.GdnDeltaArgs.from_buffer_copy(raw)
    for (name, _), v in zip(wz.GdnDeltaArgs._fields_, vals):
        assert getattr(a, name) == v, name
    assert struct.calcsize("P") == 8


def test_wrappers_refuse_wrong_tensors(wz):
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    c = cache(wz)
    with pytest.raises(ValueError):
        wz.kv_attn(q, torch.empty_like(q), c, 1, 16)  # host tensors
    with pytest.raises(ValueError):
        wz.kv_attn(q.to(torch.bfloat16), q, c, 1, 16)
    with pytest.raises(ValueError):
        wz.gdn_delta_rule(q, q, q, None, None, q, None)


@pytest.mark.parametrize("fn", ["wzyb_kv_attn_f16", "wzyb_kv_attn_f32"])
def test_attn_refuses_a_misaligned_base_position(wz, fn):
    """The kernels read it as one 4-byte word."""
    f = getattr(wz.lib(), fn)
    for at in (1, 2, 3):
        assert f(ctypes.byref(attn_args(wz, cache(wz), d_base_pos=A16 + at)), 0, None) == wz.ERR_ALIGN
    assert f(ctypes.byref(attn_args(wz, cache(wz), d_base_pos=A16 + 4)), 0, None) == wz.OK


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_no_tokens(wz, dtype):
    """No tokens are no work: an empty tensor has a null pointer, which is then no error (as in the delta rule)."""
    c, d = cache(wz), cache(wz, ring_cap=8)
    a = attn_args(wz, c, q=None, out=None, workspace=None, workspace_bytes=0)
    assert getattr(wz.lib(), f"wzyb_kv_attn_{dtype}")(ctypes.byref(a), 0, None) == wz.OK
    assert getattr(wz.lib(), f"wzyb_kv_tree_attn_{dtype}")(ctypes.byref(a), ctypes.byref(d), None, None, 0, None) == wz.OK
    empty = wz.kv_cache(*(torch.empty(0) for _ in range(4)), 0, 0)
    assert getattr(wz.lib(), f"wzyb_kv_tree_attn_{dtype}")(ctypes.byref(a), ctypes.byref(empty), None, None, 0, None) == wz.OK
    assert getattr(wz.lib(), f"wzyb_kv_attn_{dtype}")(ctypes.byref(attn_args(wz, c, q=None)), 1, None) == wz.ERR_NULL


@pytest.mark.parametrize("kh,vh,hd", [(16, 32, 128), (16, 48, 128), (2, 6, 64), (1, 1024, 128), (1024, 1024, 128)])
def test_delta_rule_workspace_of_the_largest_call_serves_shorter_ones(wz, kh, vh, hd):
    sizes = [wz.gdn_delta_rule_workspace_bytes(T, kh, vh, hd) for T in list(range(1, 4000, 7)) + list(range(4000, 70000, 333))]
    assert sizes == sorted(sizes)
    assert sizes[-1] <= 96 << 20


def test_attn_workspace_bound_for_every_length(wz):
    """The one size that the header gives for all calls."""
    worst = 0
    for qh, kvh in [(16, 2), (24, 2), (8, 2), (6, 1), (3, 3), (64, 64), (256, 1), (256, 64), (1, 1), (7, 7)]:
        for T in list(range(1, 700)) + list(range(700, 9000, 37)):
            for hd in (64, 256):
                n = wz.kv_attn_workspace_bytes(T, qh, kvh, hd)
                assert n <= 18944 * (4 * hd + 8) + 16, (T, qh, kvh, hd)
            worst = max(worst, n)
    assert worst > 18000 * (4 * 256 + 8)  # and it is not a loose one


class DeviceTensor:
    """A tensor's face on a device that need not be there."""

    def __init__(self, dtype, shape, device):
        self.dtype, self.shape, self.device_ = dtype, torch.Size(shape), device
        self.is_cuda, self.nbytes = device >= 0, 1 << 40

    def get_device(self):
        return self.device_

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return A16


class DeviceStream:
    def __init__(self, device):
        self.device_index, self.cuda_stream = device, 0x77


@pytest.fixture
def calls(wz, monkeypatch):
    """The bindings over a library that notes the device and the stream of a call; device 0 is the current one."""
    import contextlib
    import types

    now, seen = [0], []

    @contextlib.contextmanager
    def on_device(i):
        before, now[0] = now[0], i
        yield
        now[0] = before

    def entry(*args):
        seen.append((now[0], args[-1]))
        return 0

    names = [f"wzyb_{n}_{t}" for n in ("kv_attn", "kv_tree_attn", "gdn_delta_rule") for t in ("f16", "f32")]
    wz._torch_names()
    monkeypatch.setattr(wz, "lib", lambda: types.SimpleNamespace(**{n: entry for n in names}))
    monkeypatch.setattr(wz, "_current_raw_stream", lambda i: 100 + i)
    monkeypatch.setattr(wz, "_current_device", lambda: now[0], raising=False)
    monkeypatch.setattr(wz, "_on_device", on_device, raising=False)
    return seen


def mixer_calls(wz, where, stream=None):
    """One call of each binding; where(name): the device of that argument."""
    f, i, u = torch.float32, torch.int32, torch.uint8

    def t(name, dtype, *shape):
        return DeviceTensor(dtype, shape, where(name))

    kw = dict(stream=stream, workspace=t("workspace", u, 1 << 20))
    c = cache(wz)
    a = dict(lse=t("lse", f, 3, 4), d_base_pos=t("d_base_pos", i, 1), **kw)
    yield lambda: wz.kv_attn(t("q", f, 3, 4, 64), t("out", f, 3, 4, 64), c, 1, 16, **a)
    yield lambda: wz.kv_tree_attn(t("q", f, 3, 4, 64), t("out", f, 3, 4, 64), c, c, t("mask", i, 3, 1), 1, 16, t("depth", i, 3), **a)
    yield lambda: wz.gdn_delta_rule(t("q", f, 3, 2, 64), t("k", f, 3, 2, 64), t("v", f, 3, 4, 64), t("g", f, 3, 4), t("beta", f, 3, 4),
                                    t("o", f, 3, 4, 64), t("state_out", f, 4, 64, 64), state_in=t("state_in", f, 4, 64, 64),
                                    state_snaps=t("state_snaps", f, 3, 4, 64, 64), **kw)


@pytest.mark.parametrize("device", [0, 1])
def test_wrappers_launch_on_qs_device(wz, calls, device):
    for run in mixer_calls(wz, lambda name: device):
        run()
    assert calls == [(device, 100 + device)] * 3
    for run in mixer_calls(wz, lambda name: device, DeviceStream(device)):
        run()
    assert calls[3:] == [(device, 0x77)] * 3
    for run in mixer_calls(wz, lambda name: device, DeviceStream(1 - device)):
        with pytest.raises(ValueError):
            run()
    assert len(calls) == 6


@pytest.mark.parametrize("other", ["out", "lse", "d_base_pos", "workspace", "mask", "depth", "k", "v", "g", "beta", "o", "state_in",
                                   "state_out", "state_snaps"])
@pytest.mark.parametrize("device", [-1, 1])
def test_wrappers_refuse_tensors_of_two_devices(wz, calls, other, device):
    users = {"out": 2, "lse": 2, "d_base_pos": 2, "workspace": 3}.get(other, 1)
    refused = 0
    for run in mixer_calls(wz, lambda name: device if name == other else 0):
        try:
            run()
        except ValueError:
            refused += 1
    assert refused == users and len(calls) == 3 - users
