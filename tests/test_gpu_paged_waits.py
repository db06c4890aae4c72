"""The bounded waits of the attention over pages and prompts: what happens when one runs out, and when rows are slow."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from homelab_b200.backend import Gpu  # noqa: E402
from homelab_b200.paged import PagedKv  # noqa: E402

if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def gpu():
    g = Gpu(0)
    yield g
    g.set_wait_limit(0)
    torch.cuda.synchronize()
    assert g.device_error() == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def step(gpu, new, cached, fp8, H=8, K=2, D=128, page=64, seed=0):
    """One call over a pool of its own: (the call, its output, whatever it reads)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-(a + n) // page) for a, n in zip(cached, new)]
    table = torch.zeros(len(new), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    k, v = (torch.randn(at, K, page, D, generator=g, device=DEV) for _ in range(2))
    if fp8:
        e = torch.full((at, K, page), 121, dtype=torch.uint8, device=DEV)
        cache = PagedKv((k * 64).to(torch.float8_e4m3fn), (v * 64).to(torch.float8_e4m3fn), table.to(DEV), e, e.clone())
    else:
        cache = PagedKv(k.to(torch.bfloat16), v.to(torch.bfloat16), table.to(DEV))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], H, D, generator=g, device=DEV).to(torch.bfloat16)
    q_start, kv_len = i32(starts), i32([a + n for a, n in zip(cached, new)])
    out = torch.full_like(q, 5.0)

    def call():
        out.fill_(5.0)
        gpu.attention_paged(q, cache, out, q_start, kv_len, max(new), 1 / math.sqrt(D))
        return out

    return call, cache, q


PATHS = {
    "decode": ([1, 1, 1], [4000, 17, 60000]), "draft": ([4, 1], [9000, 300]), "chunk": ([300, 40], [20000, 5]),
    "many": ([200] * 40, [100] * 40), "long": ([1500], [30000]),
}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("path", PATHS)
def test_a_wait_that_runs_out_ends_the_call_with_an_error(gpu, path, fp8):
    """With next to no time to wait a call either ends as it should or sets the error word; none hangs, and the calls after it,
    the error cleared, are right again."""
    call, _, _ = step(gpu, *PATHS[path], fp8)
    want = call().clone()
    torch.cuda.synchronize()
    assert gpu.device_error() == 0
    for _ in range(3):
        try:
            gpu.set_wait_limit(1)
            out = call().clone()
            torch.cuda.synchronize()
        finally:
            gpu.set_wait_limit(0)
        code = gpu.device_error()
        assert code == 0 or code >> 4 in (0xa0, 0xb0), hex(code)
        if code == 0:
            assert torch.equal(out, want)
        assert torch.equal(call(), want)
        assert gpu.device_error() == 0
