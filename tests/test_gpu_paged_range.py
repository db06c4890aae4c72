"""Attention over e4m3 pages whose rows' powers of two lie far apart, on the GPU, against float64 (tests/paged_ref.py)."""
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
    torch.cuda.synchronize()
    assert g.device_error() == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def quantise(x):
    """x [L, K, D] as e4m3 codes and exponent bytes, as the cache's write makes them."""
    L, K, _ = x.shape
    e = torch.tensor([[R.exponent(float(x[j, h].abs().max()), 448.0) for h in range(K)] for j in range(L)])
    codes = (x.double() * torch.exp2(-e.double())[..., None]).float().to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def paged(codes_k, ke, codes_v, ve, page):
    """Rows [L, K, D] as a pool of their own with shuffled pages and a table of one sequence."""
    L, K, D = codes_k.shape
    n = -(-L // page)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(L)).to(torch.int32)
    pools = []
    for x in (codes_k.view(torch.uint8), codes_v.view(torch.uint8), ke, ve):
        full = torch.full((n * page, *x.shape[1:]), 255 if x.dim() == 2 else 0x7f, dtype=torch.uint8)  # behind the end
        full[:L] = x
        full = full.unflatten(0, (n, page)).transpose(1, 2)
        pool = torch.empty_like(full, memory_format=torch.contiguous_format)
        pool[order.long()] = full
        pools.append(pool.to(DEV))
    return PagedKv(pools[0], pools[1], order[None].to(DEV), pools[2], pools[3])


def stands_for(codes, e):
    """A row's values, as fp32 numbers: what passes fp32's range is infinite, and 0 * inf NaN."""
    return (codes.double() * torch.exp2(e.double() - 127)[..., None]).float().double()


def check(gpu, q, ck, ke, cv, ve, page, scale, n_before, score_err=0.0):
    """Attention of q's tokens behind n_before positions, within the bound of every row's own magnitudes.  On top comes what
    the three e5m2 terms of a weight leave out: half of their last unit 2^-16 at a largest weighted row of 2^11, so 2^-28 of
    that row (codes up to 448) for each position, and 2^-22 where exponents within 2^6 of one another share one reference.  An
    error of the scores counts twice, in the weight and in the sum it is divided by.  Weights below 2^-118 of a row's largest
    may be zero: exponentials end at 2^-126 in fp32, and are made 2^-8 lower."""
    n, H, D = q.shape
    L, K, _ = ck.shape
    out = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), paged(ck, ke, cv, ve, page), out, i32([0, n]), i32([L]), n, scale)
    k, v = stands_for(ck, ke), stands_for(cv, ve)
    want, mag, big = R.attend(q.double(), k, v, n_before, scale)
    _, least, _ = R.attend(q.double(), k, v.abs().clamp(max=3.4e38).amax(-1, keepdim=True).expand_as(v), n_before, scale)
    bound = R.attention_bound(want, mag, big, D) + L * 2.0 ** -22 * least
    for i in range(n):
        for h in range(H):
            x = (k[:n_before + i + 1, h // (H // K)] @ q[i, h].double()) * scale
            gone = x < x.max() - 118.0 * math.log(2.0)
            if gone.any():
                p = torch.softmax(x, 0)
                bound[i, h] += torch.where(gone[:, None] & torch.isfinite(v[:n_before + i + 1, h // (H // K)]),
                                           p[:, None] * v[:n_before + i + 1, h // (H // K)].abs(), 0.0).sum(0)
    if score_err:
        bound = bound + 2 * score_err * mag
    out = out.cpu().double()
    none = torch.isnan(want)
    assert torch.equal(torch.isnan(out), none)
    err = torch.where(out == want, 0.0, (out - want).abs())  # infinities among them
    assert (err <= bound)[~none].all(), float((err / bound)[~none].max())
    return out


def one_loud_row(L, K, D, spread, seed, where):
    """Keys and values as usual, but for position `where`: its value row is 2^spread larger, its key points away from q."""
    q = normal(seed, 1, 4 * K, D).to(torch.bfloat16)
    k, v = normal(seed + 1, L, K, D), normal(seed + 2, L, K, D)
    k[where] = -2.0 * q[0].float().unflatten(0, (K, 4)).mean(1)
    v[where] *= 2.0 ** spread
    return q, k, v


@pytest.mark.parametrize("spread", [6, 12, 18, 20, 24, 30, 60, 100])
@pytest.mark.parametrize("L,where,D", [(90, 3, 128), (1000, 0, 128), (1000, 700, 128), (1000, 999, 128), (9000, 8000, 128),
                                       (1000, 130, 64), (5000, 4999, 64)])
def test_a_visible_large_row_of_little_weight_costs_no_bits(gpu, spread, L, where, D):
    """One new token: a value row up to 2^100 larger, whose weight is too small to count, leaves the others' weights alone."""
    K = 2
    q, k, v = one_loud_row(L, K, D, spread, 17, where)
    scale = (spread + 20.0) * math.log(2.0) / float((q[0].float() ** 2).sum(-1).min()) * 4
    check(gpu, q, *quantise(k), *quantise(v), 16, scale, L - 1)


@pytest.mark.parametrize("n,H", [(1, 8), (3, 8), (4, 4), (7, 16), (16, 2), (30, 2), (200, 8)])
@pytest.mark.parametrize("spread", [18, 30, 70])
def test_large_rows_seen_by_some(gpu, n, H, spread):
    """Drafts and chunks: rows of every size among the cached positions and among the new ones, so that some query rows see a
    large one and some do not, its weight small or whole."""
    K, D, a = 2, 128, 333
    L = a + n
    q = normal(31, n, H, D).to(torch.bfloat16)
    k, v = normal(32, L, K, D), normal(33, L, K, D)
    for j in (5, 200, a, a + n // 2, L - 1):
        v[j] *= 2.0 ** spread
        if j % 2:
            k[j] = -20.0 * q[n - 1, :K].float()
    check(gpu, q, *quantise(k), *quantise(v), 32, 0.09, a)


@pytest.mark.parametrize("n,H", [(1, 8), (5, 8), (16, 2), (100, 8)])
@pytest.mark.parametrize("tiny", [1e-3, 1e-4, 1e-5, 1e-12])
@pytest.mark.parametrize("zeros", [[0], [7, 130, 131, 400], list(range(0, 420, 3))])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_zeros_among_small_values(gpu, n, H, tiny, zeros, D):
    """A row of zeros is written with exponent 0, far above the exponents of small values: it must not cost them bits."""
    K, a = 2, 420
    L = a + n
    q = normal(41, n, H, D).to(torch.bfloat16)
    k, v = normal(42, L, K, D), normal(43, L, K, D) * tiny
    v[zeros] = 0.0
    check(gpu, q, *quantise(k), *quantise(v), 64, 0.09, a)


@pytest.mark.parametrize("n,H", [(1, 8), (5, 8), (16, 2), (100, 8)])
@pytest.mark.parametrize("apart", [6, 10, 13])
@pytest.mark.parametrize("a", [2, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_queries_with_channels_of_unlike_size(gpu, n, H, apart, a, D):
    """A few channels of the queries 2^apart larger than the rest, those of the keys as much smaller: the small ones make
    most of a score.  A query's two terms are off by 2^-22 of its largest value in each channel."""
    K = 2
    L = a + n
    q, k, v = normal(91, n, H, D), normal(92, L, K, D) * 2.0, normal(93, L, K, D)
    q[..., 3::40] *= 2.0 ** apart
    k[..., 3::40] *= 2.0 ** -apart
    q = q.to(torch.bfloat16)
    ck, ke = quantise(k)
    cv, ve = quantise(v)
    more = 2.0 ** -22 * float(q.float().abs().max()) * stands_for(ck, ke).abs().sum(-1).max() * 0.09
    check(gpu, q, ck, ke, cv, ve, 16, 0.09, a, score_err=float(more))


@pytest.mark.parametrize("n,H", [(1, 8), (5, 8), (16, 2), (100, 8)])
@pytest.mark.parametrize("power", [120, 112, 95, -95, -112, -118])
def test_queries_of_any_size(gpu, n, H, power):
    """Queries near both ends of bf16's range, and a scale that brings their scores back."""
    K, D, a = 2, 128, 150
    L = a + n
    q = (normal(95, n, H, D) * 2.0 ** power).to(torch.bfloat16)
    check(gpu, q, *quantise(normal(96, L, K, D)), *quantise(normal(97, L, K, D)), 16, 0.09 * 2.0 ** -power, a)


@pytest.mark.parametrize("n,H", [(1, 8), (6, 8), (90, 8)])
@pytest.mark.parametrize("size", [300.0, 20.0, 1.0, 0.01])
@pytest.mark.parametrize("sinks,L", [([0], 400), ([0, 1, 2, 3], 3000), ([260], 300)])
def test_rows_of_zeros_that_take_the_weight(gpu, n, H, size, sinks, L):
    """Positions of zero values whose keys draw all but 2^-15 of the weight: the rest keeps its bits."""
    K, D = 2, 128
    q = normal(55, n, H, D)
    q = (q + 2.0).to(torch.bfloat16)  # a direction that all queries share
    k, v = normal(56, L, K, D), normal(57, L, K, D) * size
    k[sinks], v[sinks] = 1.0, 0.0
    scale = 15.0 * math.log(2.0) / float(q.float().sum(-1).mean())
    check(gpu, q, *quantise(k), *quantise(v), 16, scale, L - n)


def test_every_row_is_zero(gpu):
    K, D, L = 2, 128, 300
    q, k = normal(51, 1, 8, D).to(torch.bfloat16), normal(52, L, K, D)
    out = check(gpu, q, *quantise(k), *quantise(torch.zeros(L, K, D)), 16, 0.09, L - 1)
    assert not out.any()
    # and zeros in front of the first row that is none, where the others' weights are the larger ones
    v = torch.zeros(L, K, D)
    v[250:] = normal(53, 50, K, D) * 1e-6
    k[:250] = 2.0 * q[0].float().unflatten(0, (K, 4)).mean(1)
    check(gpu, q, *quantise(k), *quantise(v), 16, 0.09, L - 1)


@pytest.mark.parametrize("n,H", [(1, 8), (6, 8), (90, 8)])
@pytest.mark.parametrize("loud", [250, 245, 240, 200])
def test_exponents_over_the_whole_range(gpu, n, H, loud):
    """Bytes from 1 to 254, in pools that no append wrote: codes that do not fill their exponent among them."""
    K, D, a = 2, 128, 400
    L = a + n
    g = torch.Generator().manual_seed(61)
    q = normal(62, n, H, D).to(torch.bfloat16)
    ck, ke = quantise(normal(63, L, K, D))
    cv = (normal(64, L, K, D) * 30).to(torch.float8_e4m3fn)
    ve = torch.randint(1, 110, (L, K), generator=g, dtype=torch.uint8)
    ve[50] = loud
    ck[50] = (-q[0, :K].float() * 100).to(torch.float8_e4m3fn)  # hardly any weight
    ke[50] = 140
    check(gpu, q, ck, ke, cv, ve, 16, 0.3, a)
    cv, ve = (normal(65, L, K, D) * 30).to(torch.float8_e4m3fn), torch.full((L, K), 100, dtype=torch.uint8)
    cv[77] = (normal(66, K, D) * 2.0 ** -8).to(torch.float8_e4m3fn)  # a few units of the smallest code under a large byte
    ve[77] = 120
    check(gpu, q, ck, ke, cv, ve, 16, 0.09, a)


@pytest.mark.parametrize("n", [1, 5])
def test_large_values_do_not_pass_fp32_on_the_way(gpu, n):
    """Value rows near 2^120 over thousands of positions: their mean is an fp32 number, their sum is none."""
    K, D, a = 1, 64, 5000
    L = a + n
    q = normal(71, n, 8, D).to(torch.bfloat16)
    k, v = normal(72, L, K, D), normal(73, L, K, D)
    v = v.clamp(-3, 3) * 2.0 ** 117
    check(gpu, q, *quantise(k), *quantise(v), 64, 0.05, a)


def test_scores_of_a_billion(gpu):
    """Scores so large that an exponent added to them is rounded away: the largest takes all the weight."""
    K, D, L = 1, 128, 700
    q = torch.ones(1, 8, D).to(torch.bfloat16)
    ck = torch.full((L, K, D), 0.5).to(torch.float8_e4m3fn)
    ke = torch.full((L, K), 127, dtype=torch.uint8)
    ck[333] = 1.0
    cv, ve = quantise(normal(81, L, K, D))
    ve[::3] -= 40
    ve[333] = 90
    out = torch.empty(1, 8, D, dtype=torch.bfloat16, device=DEV)
    for scale in (1e4, 1e7, 1e12, 1e30):
        gpu.attention_paged(q.to(DEV), paged(ck, ke, cv, ve, 16), out, i32([0, 1]), i32([L]), 1, scale)
        want = stands_for(cv, ve)[333, 0].expand(8, D)
        assert ((out[0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rotated", [False, True])
def test_the_largest_finite_values_come_back_finite(gpu, src, rotated):
    """Rows that hold a type's largest values: their codes stand for fp32 numbers, off by 2^-4 of the value at most."""
    K, D, page, L = 1, 64, 16, 8
    v = normal(101, L, K, D)
    v[0, 0, 3], v[1, 0, 5] = torch.finfo(src).max, -torch.finfo(src).max
    v[2] = torch.finfo(src).max
    v[3, 0, ::2] = -torch.finfo(src).max
    v[4] *= 2.0 ** 125
    v[5, 0, 7] = 248.0 * 2.0 ** 120
    v[6, 0, 8] = 247.0 * 2.0 ** 120
    v[7, 0, 1], v[7, 0, 2] = torch.finfo(src).max, float("inf")
    v = v.to(src).to(DEV)
    cache = PagedKv.empty(2, K, page, D, i32([[1, 0]]), fp8=True)
    plan = gpu.rope_plan(16) if rotated else None  # position 0 turns by nothing
    for j in range(L):
        gpu.kv_append_paged(cache, v[j:j + 1], v[j:j + 1], i32([0, 1]), i32([1]), rope=plan)
        k_out, v_out = (torch.empty(1, K, D, dtype=torch.float32, device=DEV) for _ in range(2))
        gpu.kv_read_paged(cache, i32([0, 1]), i32([1]), k_out, v_out)
        turned = v[j].double()
        if rotated:  # 0 * inf reaches the other half of its pair
            turned = torch.from_numpy(R.rotate(v[j:j + 1].double().cpu().numpy(), [0], 16, False, *R.inv_freq(16))[0][0]).to(DEV)
        for got, want in ((k_out[0].double(), turned), (v_out[0].double(), v[j].double())):
            finite = torch.isfinite(want)
            assert torch.equal(torch.isfinite(got), finite)
            e = cache.v_exp[1, 0, 0].double() - 127
            bound = torch.maximum(2.0 ** -4 * want.abs(), torch.exp2(e - 10))
            assert ((got - want).abs() <= bound)[finite].all(), j


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 3]])
@pytest.mark.parametrize("repeat", [False, True])
def test_a_batch_of_unlike_caches_repeats_its_bits(gpu, new, repeat):
    """Sequences whose exponents lie close and far apart, side by side: right, and the same bits every time."""
    K, D, page = 2, 128, 16
    lens = [700, 130, 2500]
    rows = []
    for b, (n, L) in enumerate(zip(new, lens)):
        v = normal(112 + b, L, K, D)
        if b != 1:
            v[::7] *= 2.0 ** 25
            v[::5] = 0.0
        rows.append((*quantise(normal(110 + b, L, K, D)), *quantise(v)))
    caches = [paged(*r, page) for r in rows]
    pools = [torch.cat([getattr(c, name) for c in caches]) for name in ("k_pages", "v_pages", "k_exp", "v_exp")]
    width, at = max(c.max_pages for c in caches), 0
    table = torch.zeros(3, width, dtype=torch.int32, device=DEV)
    for b, c in enumerate(caches):
        table[b, :c.max_pages] = c.block_table[0] + at
        at += c.k_pages.shape[0]
    cache = PagedKv(pools[0], pools[1], table, pools[2], pools[3])
    q = normal(119, sum(new), 8, D).to(torch.bfloat16)
    q_start, at = [0], 0
    for n in new:
        q_start.append(q_start[-1] + n)
    out = torch.empty(sum(new), 8, D, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), cache, out, i32(q_start), i32(lens), max(new), 0.09)
    for b, (n, L) in enumerate(zip(new, lens)):
        s = slice(q_start[b], q_start[b + 1])
        k, v = stands_for(*rows[b][:2]), stands_for(*rows[b][2:])
        want, mag, big = R.attend(q[s].double(), k, v, L - n, 0.09)
        _, least, _ = R.attend(q[s].double(), k, v.abs().amax(-1, keepdim=True).expand_as(v), L - n, 0.09)
        err = (out[s].cpu().double() - want).abs()
        bound = R.attention_bound(want, mag, big, D) + L * 2.0 ** -22 * least
        assert (err <= bound).all(), (b, float((err / bound).max()))
    if repeat:
        for _ in range(20):
            again = torch.empty_like(out)
            gpu.attention_paged(q.to(DEV), cache, again, i32(q_start), i32(lens), max(new), 0.09)
            assert torch.equal(again, out)


@pytest.mark.parametrize("n,H", [(1, 8), (1, 16), (2, 8), (1, 2), (3, 4)])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("L,D", [(33, 128), (700, 128), (5000, 128), (400, 64)])
def test_few_rows_are_rounded_once(gpu, n, H, fp8, L, D):
    """Up to 8 query rows a kv head: the weights keep 15 bits (9 over e4m3 pages), so that over bf16 pages an output is the
    formula's, rounded once: 2^-8 of it; and of the magnitudes 2^-15 for the weights' terms (the first is cut off, so that the
    second is 2^-7 of the weight at most and off by 2^-8 of that), 2^-20 for what is added to the second, 2^-18 for exponentials
    and sums."""
    K, a = 2, L - n
    q = normal(131, n, H, D).to(torch.bfloat16)
    k, v = normal(132, L, K, D), normal(133, L, K, D)
    if fp8:
        check(gpu, q, *quantise(k), *quantise(v), 16, 0.09, a)
        return
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    pages = -(-L // 16)
    pool = torch.full((2, pages * 16, K, D), float("nan"), dtype=torch.bfloat16)
    pool[0, :L], pool[1, :L] = k, v
    pool = pool.unflatten(1, (pages, 16)).transpose(2, 3).contiguous().to(DEV)
    cache = PagedKv(pool[0], pool[1], torch.arange(pages, dtype=torch.int32, device=DEV)[None])
    out = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), cache, out, i32([0, n]), i32([L]), n, 0.09)
    want, mag, big = R.attend(q.double(), k.double(), v.double(), a, 0.09)
    err = (out.cpu().double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -15 + 2.0 ** -20 + 2.0 ** -18 + 4 * D * 2.0 ** -24 * big) * mag + 1e-30
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("n,H", [(1, 8), (4, 8), (16, 2), (70, 8)])
@pytest.mark.parametrize("L", [100, 900])
@pytest.mark.parametrize("spread", [40, 90, 105])
@pytest.mark.parametrize("first", [0, 20, 400])
@pytest.mark.parametrize("down", [60, 95])
def test_zeros_that_take_the_weight_beside_a_large_row(gpu, n, H, L, spread, first, down):
    """Rows of zeros draw all but 2^-down of the weight, from the start or from some position on, and a row 2^spread larger as
    little of the rest: what is left, 2^-down of the weight each, makes the output, or the large row does."""
    K, D = 2, 128
    q = (normal(141, n, H, D) + 2.0).to(torch.bfloat16)  # a direction that all queries share
    k, v = normal(142, L, K, D) * 0.2, normal(143, L, K, D)
    k[min(first, L // 2)] = 1.0
    v[min(first, L // 2)] = 0.0
    loud = L - n - 1
    k[loud], v[loud] = -1.0, v[loud] * 2.0 ** spread
    scale = down * math.log(2.0) / float(q.float().sum(-1).mean())
    check(gpu, q, *quantise(k), *quantise(v), 16, scale, L - n)
