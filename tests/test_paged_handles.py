"""Handles and workspaces of the paged cache's calls on the host: what they refuse, keep and hand on.  No GPU."""
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from homelab_b200 import backend  # noqa: E402
from homelab_b200.backend import Gpu  # noqa: E402
from homelab_b200.paged import PagedKv  # noqa: E402


def pool(pages=8, heads=2, page=16, dim=64):
    return torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16), torch.zeros(pages, heads, page, dim,
                                                                                   dtype=torch.bfloat16)


def reach(table, c):
    """The entries of the table's storage that the kernels may read: row b from b * table_stride, max_pages of them."""
    rows = [c.struct.block_table + 4 * (b * c.struct.table_stride + i) for b in range(c.batch)
            for i in range(c.struct.max_pages)]
    want = [table.data_ptr() + 4 * (b * table.stride(0) + i * table.stride(1)) for b in range(table.shape[0])
            for i in range(table.shape[1])]
    return rows, want


def test_block_table_rows_that_overlap_are_refused():
    k, v = pool()
    t = torch.arange(24, dtype=torch.int32)
    for bad in (t[:8].expand(4, 8), t[None, :8].expand(2, 8), t.as_strided((3, 8), (4, 1)), t.as_strided((2, 8), (7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            PagedKv(k, v, bad)


@pytest.mark.parametrize("table", [
    torch.arange(24, dtype=torch.int32).view(3, 8),
    torch.arange(48, dtype=torch.int32).view(3, 16)[:, 3:11],        # cut out of a wider one
    torch.arange(24, dtype=torch.int32).as_strided((2, 8), (8, 1)),  # rows back to back
    torch.arange(24, dtype=torch.int32).as_strided((1, 8), (0, 1)),  # one row: its stride leads nowhere
    torch.arange(8, dtype=torch.int32)[None].expand(1, 8),
    torch.arange(6, dtype=torch.int32)[:, None],                     # one page a sequence
    torch.arange(24, dtype=torch.int32).view(3, 8)[:, :1],
    torch.zeros(0, 5, dtype=torch.int32),
])
def test_block_table_rows_are_read_where_they_lie(table):
    k, v = pool()
    rows, want = reach(table, PagedKv(k, v, table))
    assert rows == want


class FakeLibrary:
    """The entry points that the calls below reach, on the CPU: what they were given, and a device error word."""

    def __init__(self):
        self.error, self.workspaces, self.waits = 0, [], 0.0
        self.inside, self.shared = set(), False

    def oomb_device_error(self, code, clear):
        code._obj.value = self.error
        if clear:
            self.error = 0
        return 0

    def oomb_attention_paged_workspace_bytes(self, *args):
        return 8192

    def oomb_attention_prompt_workspace_bytes(self, *args):
        return 8192

    def oomb_attention_paged(self, *args):
        self.workspaces.append(args[12])
        self.shared |= args[12] in self.inside
        self.inside.add(args[12])
        time.sleep(self.waits)  # a call's several launches
        self.inside.discard(args[12])
        return 0


@pytest.fixture
def host(monkeypatch):
    """Gpu objects that stand on the CPU, over one FakeLibrary."""
    lib = FakeLibrary()

    class Here:
        def __init__(self, *a):
            pass

        def __enter__(self):
            return self

        def __exit__(self, *a):
            return False

    monkeypatch.setattr(backend, "_current_device", lambda: -1)
    monkeypatch.setattr(backend, "_raw_stream", lambda i: 77)
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    monkeypatch.setattr(backend.torch.cuda, "device", Here)
    monkeypatch.setattr(backend._lib, "lib", lambda: lib)
    monkeypatch.setattr(backend.torch, "device", lambda *a: torch.empty(0).device)

    def make():
        g = Gpu(-1)
        assert g.L is lib
        return g

    return lib, make


def attend(g):
    k, v = pool(dim=128)
    cache = PagedKv(k, v, torch.zeros(2, 3, dtype=torch.int32))
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    g.attention_paged(x, cache, x.clone(), None, torch.ones(2, dtype=torch.int32), 1, 0.1)


def counters(g):
    """The words that have to be zero, of the workspace that the object keeps."""
    return next(w for k, w in g._attn_ws.items() if isinstance(k, int))[:backend._lib.ATTENTION_ZERO_BYTES]


def test_kept_workspaces_are_zero_again_after_a_device_error(host):
    lib, make = host
    g, other = make(), make()
    attend(g), attend(other)
    attend(g)
    assert lib.workspaces[0] == lib.workspaces[2] != lib.workspaces[1], "one is kept"
    for x in (g, other):
        counters(x)[5] = 1  # an arrival that the call which gave up left behind
    lib.error = 0xb06
    assert g.device_error() == 0xb06
    attend(g), attend(other)
    assert not counters(g).any() and not counters(other).any()
    kept = counters(g)
    assert g.device_error() == 0
    attend(g)
    assert counters(g).data_ptr() == kept.data_ptr(), "without an error nothing is made anew"


def test_threads_on_one_stream_take_turns(host):
    """Two threads' calls over one kept workspace: the launches of one do not come between those of the other."""
    lib, make = host
    g = make()
    attend(g)
    lib.waits = 0.005
    threads = [threading.Thread(target=lambda: [attend(g) for _ in range(5)]) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(lib.workspaces) == 21 and len(set(lib.workspaces)) == 1
    assert not lib.shared


# ---- operands that share memory: refused before any launch ----------------------------------

HERE = 1 << 20  # an address that is never followed


@pytest.mark.parametrize("x,sx,y,sy,t,meet", [
    (0, 512, 3 * 1024, 512, 3, False),      # one behind the other (bytes apart; strides in elements of 2 bytes)
    (0, 512, 3 * 1024 - 16, 512, 3, True),
    (0, 512, 1024, 512, 3, True),           # shifted by a token
    (0, 512, -2 * 1024, 512, 3, True),
    (0, 512, -3 * 1024, 512, 3, False),
    (0, 512, 16, 512, 3, True),
    (0, 1024, 1024, 1024, 3, False),        # side by side in rows of 2,048 bytes
    (0, 1024, 1024 - 16, 1024, 3, True),
    (1024, 1024, 0, 1024, 3, False),
    (1024, 1024, 2 * 2048, 1024, 3, False),
    (1024, 1024, 2 * 2048 + 16, 1024, 3, True),
    (0, 512, 1024, 1024, 1, False),         # a single row has no stride
    (0, 512, 1024 - 16, 1024, 1, True),
    (0, 512, 2048, 1024, 4, True),          # unlike strides in one stretch
    (0, 512, 0, 512, 0, False),
])
def test_operands_that_share_memory_are_refused(x, sx, y, sy, t, meet):
    """Rows of 8 heads of 64 bf16 values, 1,024 bytes."""
    import ctypes as C

    from homelab_b200 import _lib
    L = _lib.lib()
    far = HERE + (1 << 24)
    X, Y = HERE + x, HERE + y
    passes = (0,) if t == 0 else (_lib.E_DEVICE,)  # all checks passed: nothing to do, or no device here
    if torch.cuda.is_available():
        pytest.skip("calls that pass their checks would launch")
    want = (_lib.E_ARG,) if meet else passes
    rope = C.byref(_lib.RopeStruct(rot_dim=64, interleaved=0, mscale=1.0, turns=far))
    cache = C.byref(_lib.PagedKvStruct(dtype=0, kv_heads=8, head_dim=64, page_size=16, num_pages=10, max_pages=4, table_stride=4,
                                       k=far, v=far, page_stride=8 * 16 * 64, block_table=far))
    assert L.oomb_rope_rows(rope, X, 1, sx, far, Y, sy, t, 8, 64, None) in want
    B = t
    assert L.oomb_attention_paged(cache, X, sx, Y, sy, 8, None, far, B, t, 1, 0.1, far, 1 << 40, None) in want
    # queries, keys or values of a prompt under its output
    for a in range(3):
        rows = [(far + (1 << 22) * i, 512) for i in range(3)]
        rows[a] = (X, sx)
        (q, qs), (k, ks), (v, vs) = rows
        assert L.oomb_attention_prompt(q, qs, k, ks, v, vs, Y, sy, 8, 8, 64, far, 1, t, 1, 0.1, far, 1 << 40, None) in want, a
        assert L.oomb_kv_append_paged(cache, rope, q, qs, Y, sy, 8, k, ks, v, vs, 1, None, far, B, t, None) in want, a
    if sx == sy:
        assert L.oomb_kv_read_paged(cache, None, far, B, t, X, Y, 1, sx, None) in want


def test_operations_in_place():
    import ctypes as C

    from homelab_b200 import _lib
    if torch.cuda.is_available():
        pytest.skip("calls that pass their checks would launch")
    L = _lib.lib()
    far = HERE + (1 << 24)
    rope = C.byref(_lib.RopeStruct(rot_dim=64, interleaved=0, mscale=1.0, turns=far))
    cache = C.byref(_lib.PagedKvStruct(dtype=0, kv_heads=8, head_dim=64, page_size=16, num_pages=10, max_pages=4, table_stride=4,
                                       k=far, v=far, page_stride=8 * 16 * 64, block_table=far))
    assert L.oomb_rope_rows(rope, HERE, 0, 512, far, HERE, 512, 3, 8, 64, None) == _lib.E_DEVICE
    assert L.oomb_rope_rows(rope, HERE, 0, 512, far, HERE, 520, 3, 8, 64, None) == _lib.E_ARG  # the same rows, another stride
    append = lambda dt, qs, qos, qo: L.oomb_kv_append_paged(  # noqa: E731
        cache, rope, HERE, qs, qo, qos, 8, HERE + 1024, 1536, HERE + 2048, 1536, dt, None, far, 3, 3, None)
    assert append(1, 1536, 1536, HERE) == _lib.E_DEVICE   # the queries of a fused projection's rows, in place
    assert append(1, 1536, 1544, HERE) == _lib.E_ARG
    assert append(1, 1536, 1536, HERE + 1024) == _lib.E_ARG  # over the keys
    assert L.oomb_kv_append_paged(cache, rope, HERE, 1536, HERE, 3080, 8, HERE + 2048, 1536, HERE + 4096, 1536, 0, None, far, 3, 3,
                                  None) == _lib.E_ARG     # fp32 rows are not written over in bf16
