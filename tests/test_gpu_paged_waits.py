"""The bounded waits of the attention over pages and prompts: what happens when one runs out, and when rows are slow."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import paged_ref as R  # noqa: E402
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


def exact(cache, q, b, at, n, a, scale):
    """The rows of sequence b in float64 on the GPU, a head at a time, and the bound of their error."""
    K, D, L = cache.kv_heads, cache.head_dim, a + n
    ids = cache.block_table[b, :-(-L // cache.page_size)].long()
    k, v = (x[ids].double().transpose(1, 2).flatten(0, 1)[:L] for x in (cache.k_pages, cache.v_pages))
    if cache.fp8:
        k, v = (x * torch.exp2(e[ids].double() - 127).transpose(1, 2).flatten(0, 1)[:L][..., None]
                for x, e in ((k, cache.k_exp), (v, cache.v_exp)))
    later = torch.arange(L, device=DEV)[None] > torch.arange(a, a + n, device=DEV)[:, None]
    x = q[at:at + n].double()
    H = x.shape[1]
    out, mag, big = (torch.empty(n, H, d, dtype=torch.float64, device=DEV) for d in (D, D, 1))
    for h in range(H):
        kk, vv = k[:, h // (H // K)], v[:, h // (H // K)]
        p = (x[:, h] @ kk.T * scale).masked_fill(later, float("-inf")).softmax(-1)
        seen = torch.where(torch.isfinite(vv), vv, 0.0)  # what is hidden has no weight
        out[:, h], mag[:, h] = p @ seen, p @ seen.abs()
        big[:, h, 0] = (x[:, h].abs() @ kk.abs().T).masked_fill(later, 0.0).amax(-1) * abs(scale)
    return out, R.attention_bound(out, mag, big, D)


def plant(cache, b, j):
    """A value that is not finite at position j of sequence b, in every kv head's dimension 7."""
    page, slot = int(cache.block_table[b, j // cache.page_size]), j % cache.page_size
    v = cache.v_pages.view(torch.uint8) if cache.fp8 else cache.v_pages
    v[page, :, slot, 7] = 0x7f if cache.fp8 else float("inf")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached", [([300, 40], [60000, 5]), ([100, 20], [60000, 5]), ([4] * 30, [9000] * 30)])
def test_a_visible_value_that_is_not_finite_costs_nothing(gpu, fp8, new, cached):
    """Position 0 of the first sequence: its rows are what the arithmetic makes of it, at once, and the others are as ever."""
    call, cache, _ = step(gpu, new, cached, fp8, seed=3)
    want = call().clone()
    plant(cache, 0, 0)
    try:
        gpu.set_wait_limit(2_000_000)  # 2 ms: one warp over 32 rows of 60,000 positions takes some 150
        got = call().clone()
        torch.cuda.synchronize()
    finally:
        gpu.set_wait_limit(0)
    assert gpu.device_error() == 0
    n = new[0]
    assert torch.equal(got[n:], want[n:])
    hit = got[:n, :, 7].float()
    assert (torch.isnan(hit) if fp8 else torch.isnan(hit) | torch.isinf(hit)).all()
    others = [d for d in range(128) if d != 7]
    assert torch.equal(got[:n][..., others], want[:n][..., others])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached", [([300, 40], [60000, 5]), ([100, 20], [60000, 5]), ([4, 4], [200000, 3])])
def test_rows_that_are_done_again_outlast_the_waits(gpu, fp8, new, cached):
    """A value that is not finite at the last new token: rows of its tile are done again over the whole cache, which takes far
    longer than the limit, while the other warps wait."""
    call, cache, q = step(gpu, new, cached, fp8, seed=5)
    n, a = new[0], cached[0]
    want, bound = exact(cache, q, 0, 0, n, a, 1 / math.sqrt(128))
    clean = call().clone()
    plant(cache, 0, a + n - 1)
    try:
        gpu.set_wait_limit(2_000_000)
        got = call().clone()
        torch.cuda.synchronize()
    finally:
        gpu.set_wait_limit(0)
    assert gpu.device_error() == 0
    assert torch.equal(got[n:], clean[n:])
    err = (got[:n - 1].double() - want[:n - 1]).abs()
    assert (err <= bound[:n - 1]).all(), float((err / bound[:n - 1]).max())
    hit = got[n - 1, :, 7].float()
    assert (torch.isnan(hit) if fp8 else hit == float("inf")).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 5, 60, 200])
@pytest.mark.parametrize("rising", [False, True])
def test_sums_of_large_values_stay_in_range(gpu, fp8, n, rising):
    """Values of 2^112 whose weights may stand 2^8 above one while a maximum lags behind: 2,000 of them pass fp32's range
    unless the weights are held lower."""
    call, cache, q = step(gpu, [n], [2000], fp8, seed=7)
    if fp8:
        cache.v_exp.fill_(121 + 112)
    else:
        cache.v_pages.mul_(2.0 ** 112)
    if rising:  # scores that grow along the cache, by less than the 2^8 (2^4) that a maximum may lag behind a tile
        ramp = torch.arange(cache.k_pages.shape[0] * cache.page_size, device=DEV).view(-1, 1, cache.page_size, 1) / 2200.0
        q.copy_(q.abs())
        k = cache.k_pages.float() * 0.1 + ramp * (28.0 if fp8 else 0.5)
        cache.k_pages.copy_(k.to(cache.k_pages.dtype))
    got = call()
    want, bound = exact(cache, q, 0, 0, n, 2000, 1 / math.sqrt(128))
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached", [([1, 2], [300, 40]), ([5, 3], [300, 2]), ([200, 9], [77, 300]), ([70, 40], [1000, 5])])
@pytest.mark.parametrize("at", list(range(0, 32, 3)) + [129])
def test_a_key_that_is_not_finite_makes_its_rows_nan(gpu, fp8, new, cached, at):
    """At any position of a tile, with no value beside it that is not finite: every row of its kv head that sees it is NaN, the
    other kv head's and the other sequence's rows are as ever."""
    call, cache, _ = step(gpu, new, cached, fp8, seed=9)
    want = call().clone()
    page, slot = int(cache.block_table[0, at // cache.page_size]), at % cache.page_size
    for bad in ((0x7f,) if fp8 else (float("nan"), float("inf"))):
        k = cache.k_pages.view(torch.uint8) if fp8 else cache.k_pages
        keep = k[page, 1, slot, 5].clone()
        k[page, 1, slot, 5] = bad
        got = call().clone()
        k[page, 1, slot, 5] = keep
        n, first = new[0], max(0, at - cached[0])  # the first new token that sees it
        assert torch.equal(got[n:], want[n:]) and torch.equal(got[:n, :4], want[:n, :4])
        assert torch.equal(got[:min(first, n), 4:], want[:min(first, n), 4:])
        rows = got[first:n, 4:]
        if bad == float("inf"):  # a score of +inf makes NaN, one of -inf no weight
            q = step(gpu, new, cached, fp8, seed=9)[2][first:n, 4:, 5]
            up = q > 0
            assert torch.isnan(rows[up]).all() and torch.isfinite(rows[q < 0].float()).all()
        else:
            assert torch.isnan(rows).all()


@pytest.mark.parametrize("at", list(range(0, 32, 3)) + [129])
def test_a_key_of_a_prompt_that_is_not_finite(gpu, at):
    H, K, D, n = 8, 2, 128, 200
    g = torch.Generator(device=DEV).manual_seed(11)
    q, k, v = (torch.randn(n + 30, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (H, K, K))
    want, got = torch.empty_like(q), torch.empty_like(q)
    gpu.attention_prompt(q, k, v, want, i32([0, n, n + 30]), n, 0.09)
    k[at, 1, 7] = float("nan")
    gpu.attention_prompt(q, k, v, got, i32([0, n, n + 30]), n, 0.09)
    assert torch.isnan(got[at:n, 4:]).all()
    assert torch.equal(got[:, :4], want[:, :4]) and torch.equal(got[:at], want[:at]) and torch.equal(got[n:], want[n:])
