"""Rotary frequencies, and the refusals of the paged cache's calls: checked without a GPU, before any launch."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import homelab_b200 as hb  # noqa: E402
import paged_ref as R  # noqa: E402
from homelab_b200 import _lib  # noqa: E402
from homelab_b200.backend import Gpu  # noqa: E402
from homelab_b200.paged import PagedKv, RopePlan, rope_turns  # noqa: E402

FAKE = 0x10000  # never dereferenced: every call below fails its checks first


@pytest.mark.parametrize("rot", [16, 64, 96, 128])
@pytest.mark.parametrize("args", [(10000.0, "none", 1.0, 0), (500000.0, "linear", 4.0, 0), (10000.0, "ntk", 8.0, 0),
                                  (500000.0, "by_parts", 16.0, 8192), (10000.0, "by_parts", 1.0, 4096)])
def test_turns_are_the_frequencies(rot, args):
    turns, m = rope_turns(rot, *args)
    inv, want_m = R.inv_freq(rot, *args)
    got = [(int(t) % 2 ** 64) / 2.0 ** 64 * 2 * math.pi for t in turns]
    assert len(got) == rot // 2
    # float64 powers and logarithms on the other side (a few of its roundings), and half a unit of 2^-64 turns:
    # 2 pi 2^-65 of an angle, which is 6.6e-14 of the least frequency here (2.6e-6)
    assert all(abs(g - w) <= 2e-14 * w + 2 * math.pi * 2.0 ** -65 for g, w in zip(got, inv))
    assert abs(m - want_m) <= 2 ** -24 * want_m


def test_turns_refusals():
    L = hb.lib()
    m = C.c_float()
    buf = (C.c_uint64 * 64)()
    ok = (128, 10000.0, 0, 1.0, 0)
    assert L.oomb_rope_turns(*ok, buf, C.byref(m)) == 0
    for bad, status in [((24, 1e4, 0, 1.0, 0), _lib.E_SHAPE), ((0, 1e4, 0, 1.0, 0), _lib.E_SHAPE),
                        ((144, 1e4, 0, 1.0, 0), _lib.E_SHAPE), ((128, 1.0, 0, 1.0, 0), _lib.E_ARG),
                        ((128, float("nan"), 0, 1.0, 0), _lib.E_ARG), ((128, 1e4, 4, 1.0, 0), _lib.E_ARG),
                        ((128, 1e4, -1, 1.0, 0), _lib.E_ARG), ((128, 1e4, 1, 0.5, 0), _lib.E_ARG),
                        ((128, 1e4, 3, 2.0, 0), _lib.E_ARG), ((128, 1e4, 1, float("inf"), 0), _lib.E_ARG)]:
        assert L.oomb_rope_turns(*bad, buf, C.byref(m)) == status, bad
    assert L.oomb_rope_turns(*ok, None, C.byref(m)) == _lib.E_ARG
    with pytest.raises(ValueError):
        rope_turns(128, scaling="other")
    with pytest.raises(hb.OombError):
        rope_turns(24)


def struct(**kw):
    c = dict(dtype=0, kv_heads=8, head_dim=128, page_size=16, num_pages=10, max_pages=4, table_stride=4, k=FAKE, v=FAKE,
             k_exp=None, v_exp=None, page_stride=8 * 16 * 128, exp_page_stride=0, block_table=FAKE)
    c.update(kw)
    return _lib.PagedKvStruct(**c)


BAD_CACHES = [
    (dict(dtype=2), _lib.E_ARG), (dict(k=None), _lib.E_ARG), (dict(block_table=None), _lib.E_ARG),
    (dict(kv_heads=0), _lib.E_SHAPE), (dict(head_dim=96), _lib.E_SHAPE), (dict(head_dim=256), _lib.E_SHAPE),
    (dict(page_size=8), _lib.E_SHAPE), (dict(page_size=48), _lib.E_SHAPE), (dict(page_size=256), _lib.E_SHAPE),
    (dict(num_pages=0), _lib.E_SHAPE), (dict(max_pages=-1), _lib.E_SHAPE), (dict(table_stride=3), _lib.E_SHAPE),
    (dict(page_stride=8 * 16 * 128 - 8), _lib.E_SHAPE), (dict(page_stride=8 * 16 * 128 + 4), _lib.E_ALIGN),
    (dict(k=FAKE + 8), _lib.E_ALIGN), (dict(block_table=FAKE + 2), _lib.E_ALIGN),
    (dict(max_pages=1 << 27, table_stride=1 << 27), _lib.E_SHAPE),
    (dict(dtype=1), _lib.E_ARG), (dict(dtype=1, k_exp=FAKE, v_exp=FAKE), _lib.E_SHAPE),
    (dict(dtype=1, k_exp=FAKE, v_exp=FAKE, exp_page_stride=136), _lib.E_ALIGN),
    (dict(dtype=1, k_exp=FAKE + 1, v_exp=FAKE, exp_page_stride=128), _lib.E_ALIGN),
]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_every_call_checks_the_cache(kw, status):
    L = hb.lib()
    c = C.byref(struct(**kw))
    assert L.oomb_kv_append_paged(c, None, None, 0, None, 0, 0, FAKE, 1024, FAKE, 1024, 1, FAKE, FAKE, 1, 1, None) == status
    assert L.oomb_kv_read_paged(c, FAKE, FAKE, 1, 1, FAKE, FAKE, 1, 1024, None) == status
    assert L.oomb_attention_paged(c, FAKE, 4096, FAKE, 4096, 32, FAKE, FAKE, 1, 1, 1, 1.0, FAKE, 1 << 30, None) == status


def test_append_refusals():
    L = hb.lib()
    ok = dict(c=C.byref(struct()), rope=None, q=None, qs=0, qo=None, qos=0, heads=0, k=FAKE, ks=1024, v=FAKE, vs=1024, dt=1,
              q_start=FAKE, kv_len=FAKE, batch=2, t=3)

    def call(**kw):
        return L.oomb_kv_append_paged(*{**ok, **kw}.values(), None)

    rope = _lib.RopeStruct(rot_dim=128, interleaved=0, mscale=1.0, turns=FAKE)
    assert call(c=None) == _lib.E_ARG
    assert call(k=None) == _lib.E_ARG
    assert call(kv_len=None) == _lib.E_ARG
    assert call(dt=2) == _lib.E_ARG
    assert call(batch=-1) == _lib.E_SHAPE
    assert call(q_start=None) == _lib.E_SHAPE  # one token a sequence: batch == t
    assert call(ks=1016) == _lib.E_SHAPE       # rows would overlap
    assert call(vs=1028) == _lib.E_ALIGN
    assert call(k=FAKE + 8) == _lib.E_ALIGN
    assert call(q=FAKE, qs=4096, heads=32) == _lib.E_ARG  # q without q_out
    assert call(q=FAKE, qs=4096, qo=FAKE, qos=4096, heads=0) == _lib.E_SHAPE
    assert call(q=FAKE, qs=4096, qo=FAKE, qos=4088, heads=32) == _lib.E_SHAPE
    assert call(rope=C.byref(_lib.RopeStruct(rot_dim=24, mscale=1.0, turns=FAKE))) == _lib.E_SHAPE
    assert call(rope=C.byref(_lib.RopeStruct(rot_dim=144, mscale=1.0, turns=FAKE))) == _lib.E_SHAPE
    assert call(rope=C.byref(_lib.RopeStruct(rot_dim=128, mscale=0.0, turns=FAKE))) == _lib.E_ARG
    assert call(rope=C.byref(_lib.RopeStruct(rot_dim=128, mscale=1.0, turns=None))) == _lib.E_ARG
    assert call(rope=C.byref(rope), t=0) == 0  # nothing to do
    assert call(batch=0) == 0


def test_rope_read_and_attention_refusals():
    L = hb.lib()
    rope = _lib.RopeStruct(rot_dim=64, interleaved=1, mscale=1.0, turns=FAKE)
    r = C.byref(rope)
    assert L.oomb_rope_rows(None, FAKE, 1, 512, FAKE, FAKE, 512, 1, 8, 64, None) == _lib.E_ARG
    assert L.oomb_rope_rows(r, FAKE, 1, 512, None, FAKE, 512, 1, 8, 64, None) == _lib.E_ARG
    assert L.oomb_rope_rows(r, FAKE, 1, 512, FAKE, FAKE, 512, 1, 8, 80, None) == _lib.E_SHAPE
    assert L.oomb_rope_rows(r, FAKE, 1, 504, FAKE, FAKE, 512, 1, 8, 64, None) == _lib.E_SHAPE
    assert L.oomb_rope_rows(r, FAKE, 0, 514, FAKE, FAKE, 512, 1, 8, 64, None) == _lib.E_ALIGN
    assert L.oomb_rope_rows(r, FAKE, 1, 512, FAKE, FAKE, 512, 0, 8, 64, None) == 0
    c = C.byref(struct())
    assert L.oomb_kv_read_paged(c, FAKE, FAKE, 1, 1, FAKE, None, 1, 1024, None) == _lib.E_ARG
    assert L.oomb_kv_read_paged(c, FAKE, FAKE, 1, 1, FAKE, FAKE, 1, 1000, None) == _lib.E_SHAPE
    assert L.oomb_kv_read_paged(c, None, FAKE, 2, 1, FAKE, FAKE, 1, 1024, None) == _lib.E_SHAPE
    ok = dict(c=c, q=FAKE, qs=4096, out=2 * FAKE, os=4096, heads=32, q_start=FAKE, kv_len=FAKE, batch=2, t=3, max_q=2,
              scale=0.1, ws=FAKE, n=1 << 30)

    def call(**kw):
        return L.oomb_attention_paged(*{**ok, **kw}.values(), None)

    assert call(q=None) == _lib.E_ARG
    assert call(ws=None) == _lib.E_ARG
    assert call(scale=float("nan")) == _lib.E_ARG
    assert call(scale=-3e38) == _lib.E_ARG
    assert call(heads=30) == _lib.E_SHAPE       # heads % kv_heads
    assert call(heads=8 * 65, qs=1 << 20, os=1 << 20) == _lib.E_SHAPE
    assert call(qs=4088) == _lib.E_SHAPE
    assert call(qs=4100) == _lib.E_ALIGN
    assert call(out=FAKE + 2) == _lib.E_ALIGN
    assert call(max_q=-1) == _lib.E_SHAPE
    assert call(q_start=None) == _lib.E_SHAPE
    assert call(out=FAKE, q=FAKE) == _lib.E_ARG  # the output over the queries
    assert call(ws=FAKE + 16) == _lib.E_ALIGN
    assert call(t=0) == 0
    assert call(max_q=0) == 0
    p = dict(q=FAKE, qs=4096, k=FAKE, ks=1024, v=FAKE, vs=1024, out=2 * FAKE, os=4096, heads=32, kv_heads=8, d=128, q_start=FAKE,
             batch=2, t=3, max_q=2, scale=0.1, ws=FAKE, n=1 << 30)

    def prompt(**kw):
        return L.oomb_attention_prompt(*{**p, **kw}.values(), None)

    assert prompt(q_start=None) == _lib.E_ARG
    assert prompt(k=None) == _lib.E_ARG
    assert prompt(ks=1000) == _lib.E_SHAPE
    assert prompt(vs=1028) == _lib.E_ALIGN
    assert prompt(d=96) == _lib.E_SHAPE
    assert prompt(kv_heads=0) == _lib.E_SHAPE
    assert prompt(out=FAKE) == _lib.E_ARG
    assert prompt(k=2 * FAKE) == _lib.E_ARG  # the output over the keys
    assert prompt(ws=FAKE + 16) == _lib.E_ALIGN
    assert prompt(batch=0) == 0


def test_handles_refuse_what_does_not_fit():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.int32)
    c = PagedKv(k, k.clone(), t)
    assert (c.struct.num_pages, c.struct.page_stride, c.struct.max_pages) == (4, 2 * 16 * 64, 3)
    both = torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16)  # keys and values of a page side by side
    assert PagedKv(both[:, 0], both[:, 1], t).struct.page_stride == 2 * 2 * 16 * 64
    with pytest.raises(TypeError):
        PagedKv(k.float(), k.float(), t)
    with pytest.raises(ValueError):
        PagedKv(k, k[:3], t)
    with pytest.raises(ValueError):
        PagedKv(k.transpose(1, 2), k.transpose(1, 2), t)
    with pytest.raises(ValueError):
        PagedKv(k, k.clone(), t.long())
    with pytest.raises(ValueError):
        PagedKv(k, k.clone(), t.t())
    codes, e = torch.zeros(4, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, 16, dtype=torch.uint8)
    assert PagedKv(codes, codes.clone(), t, e, e.clone()).fp8
    with pytest.raises(TypeError):
        PagedKv(k, k.clone(), t, e, e.clone())
    with pytest.raises(ValueError):
        PagedKv(codes, codes.clone(), t, e)
    with pytest.raises(ValueError):
        PagedKv(codes, codes.clone(), t, e, e[:, :1])


def test_methods_refuse_what_lives_elsewhere():
    """A Gpu object that stands on the CPU: every call fails before a launch."""
    g = Gpu.__new__(Gpu)
    g.device, g.index, g.L, g._attn_ws = torch.device("cpu"), -1, hb.lib(), {}
    plan = RopePlan("cpu", 128)
    plan.index = 3
    x, pos = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="frequencies"):
        g.rope(x, pos, plan)
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    cache = PagedKv(k, k.clone(), torch.zeros(2, 3, dtype=torch.int32))
    kv = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="frequencies"):
        g.kv_append_paged(cache, kv, kv, None, pos, rope=plan)
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    for bad in (ws.view(torch.int32), ws[:64].expand(4, 64), ws[::2]):
        with pytest.raises(ValueError, match="workspace"):
            g.attention_paged(x, cache, x.clone(), None, pos, 1, 0.1, workspace=bad)
        with pytest.raises(ValueError, match="workspace"):
            g.attention_prompt(x, kv, kv, x.clone(), torch.tensor([0, 2], dtype=torch.int32), 2, 0.1, workspace=bad)
    with pytest.raises(ValueError, match="q_start"):
        g.attention_prompt(x, kv, kv, x.clone(), None, 2, 0.1)
