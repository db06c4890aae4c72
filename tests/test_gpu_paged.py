"""Rotary positions, the paged cache and the attention over it on the GPU, against float64 (tests/paged_ref.py)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import paged_ref as R  # noqa: E402
from homelab_b200.backend import Gpu  # noqa: E402
from homelab_b200.paged import PagedKv  # noqa: E402

if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

DEV = torch.device("cuda", 0)
ERR_KV_TABLE, ERR_KV_SEQ = 0x900, 0x910
SCALINGS = {"none": (10000.0, "none", 1.0, 0), "linear": (10000.0, "linear", 4.0, 0), "ntk": (10000.0, "ntk", 8.0, 0),
            "by_parts": (500000.0, "by_parts", 16.0, 8192)}


@pytest.fixture(scope="module")
def gpu():
    g = Gpu(0)
    yield g
    torch.cuda.synchronize()
    assert g.device_error() == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def normal(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * scale


class Batch:
    """A pool with random content and a shuffled block table for sequences of the given lengths."""

    def __init__(self, seed, q_start, kv_len, kv_heads, D, page, fp8, fill=None, spare=2):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in kv_len]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.zeros((len(kv_len), max(need + [1])), dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_cpu, self.pages = table, pages
        both = normal(seed + 1, pages, 2, kv_heads, page, D)  # keys and values of a page side by side
        if fp8:
            e = torch.randint(122, 126, (2, pages, kv_heads, page), generator=g, dtype=torch.uint8)
            codes = (both * 32).to(torch.float8_e4m3fn).view(torch.uint8)
            pool = codes.to(DEV)
            k, v, ke, ve = pool[:, 0], pool[:, 1], e[0].to(DEV), e[1].to(DEV)
        else:
            pool = both.to(torch.bfloat16).to(DEV)
            k, v, ke, ve = pool[:, 0], pool[:, 1], None, None
        self.pool = pool
        self.kv_heads, self.D, self.page, self.fp8 = kv_heads, D, page, fp8
        self.q_start_list, self.kv_len_list = list(q_start), list(kv_len)
        self.cache = PagedKv(k, v, table.to(DEV), ke, ve)
        self.q_start, self.kv_len = i32(q_start), i32(kv_len)

    def values(self):
        c = self.cache
        return R.values(c.k_pages, c.k_exp), R.values(c.v_pages, c.v_exp)

    def poison_unused(self):
        """NaN in every slot that no sequence uses, the tails of the last pages among them."""
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for b, n in enumerate(self.kv_len_list):
            for j in range(n):
                used[self.table_cpu[b, j // self.page], j % self.page] = True
        free = (~used).to(DEV)
        for x in (self.cache.k_pages, self.cache.v_pages):
            x.transpose(1, 2)[free] = 0x7f if self.fp8 else float("nan")


# ---- rotation ----------------------------------------------------------------------------


@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (128, 48, False),
                                               (128, 16, True), (64, 64, False), (64, 32, True), (64, 16, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,scaling", [(1, 1, "none"), (7, 5, "by_parts"), (701, 3, "linear"), (33, 32, "ntk")])
def test_rope_matches_float64(gpu, D, rot, interleaved, dtype, T, H, scaling):
    plan = gpu.rope_plan(rot, *SCALINGS[scaling], interleaved=interleaved)
    wide = normal(T + D + rot, T, H + 2, D).to(dtype).to(DEV)
    x = wide[:, 1:1 + H]  # rows inside wider ones
    pos = [int(v) for v in np.random.default_rng(T).integers(-5, 4_000_000, T)]
    pos[0] = 0 if T == 1 else 131071
    inv, m = R.inv_freq(rot, *SCALINGS[scaling])
    want, mag = R.rotate(x.cpu().double().numpy(), pos, rot, interleaved, inv, m)
    bound = R.ROPE_ERR * mag + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0) + 1e-30
    got = gpu.rope(x, i32(pos), plan)
    err = np.abs(got.cpu().double().numpy() - want)
    assert (err <= bound).all(), (err / bound).max()
    before = wide.clone()
    gpu.rope(x, i32(pos), plan, out=x)  # in place
    assert torch.equal(x, got)
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, -1], before[:, -1])


def test_rope_refuses(gpu):
    plan = gpu.rope_plan(128)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError):
        gpu.rope(x.half(), i32([0, 1, 2]), plan)
    with pytest.raises(ValueError):
        gpu.rope(x, i32([0, 1]), plan)
    with pytest.raises(ValueError):
        gpu.rope(x, torch.zeros(3, dtype=torch.int64, device=DEV), plan)
    with pytest.raises(ValueError):
        gpu.rope(x.transpose(0, 1), i32([0, 1]), plan)
    with pytest.raises(Exception):
        gpu.rope(torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV), i32([0, 1, 2]), plan)  # rot_dim > D
    with pytest.raises(TypeError):
        gpu.rope(x, i32([0, 1, 2]), plan, out=x.float())
    assert gpu.rope(x[:0], i32([]), plan).shape == (0, 2, 128)


# ---- append and read-back -----------------------------------------------------------------


def append_case(gpu, seed, new, cached, H, K, D, page, fp8, src, scaling, rot, interleaved, behind=3):
    """Appends a packed step out of fused rows with `behind` rows after the last sequence; checks all of it."""
    q_start = [0]
    for n in new:
        q_start.append(q_start[-1] + n)
    T = q_start[-1] + behind
    kv_len = [a + n for a, n in zip(cached, new)]
    B = Batch(seed, q_start, kv_len, K, D, page, fp8)
    rows = normal(seed + 5, T, (H + 2 * K) * D)
    rows[: T // 3] *= 2.0 ** -20  # rows of very unlike sizes
    rows[T // 2:, H * D:] *= 300.0
    if T > 4:
        rows[3, H * D:] = 0.0
    rows = rows.to(src).to(DEV)
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    plan = gpu.rope_plan(rot, *SCALINGS[scaling], interleaved=interleaved) if scaling else None
    inv, m = R.inv_freq(rot, *SCALINGS[scaling]) if scaling else (None, 1.0)
    pool, exps = B.pool.clone(), [None if x is None else x.clone() for x in (B.cache.k_exp, B.cache.v_exp)]
    q_out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    gpu.kv_append_paged(B.cache, k, v, B.q_start, B.kv_len, rope=plan, q=q, q_out=q_out)
    torch.cuda.synchronize()
    at = list(R.places(q_start, kv_len, page))
    tok, pos = [a[0] for a in at], [a[2] for a in at]
    page_of = [int(B.table_cpu[b, p // page]) for _, b, p in at]
    slot = [p % page for p in pos]
    q64, k64, v64 = (x[tok].cpu().double().numpy() for x in (q, k, v))
    if scaling:
        (wq, mq), (wk, mk) = (R.rotate(x, pos, rot, interleaved, inv, m) for x in (q64, k64))
    else:
        wq, mq, wk, mk = q64, 0 * q64, k64, 0 * k64
    got_q = q_out[tok].cpu().double().numpy()
    assert (np.abs(got_q - wq) <= R.ROPE_ERR * mq + 2.0 ** -8 * np.abs(wq) + 1e-38).all()
    if behind:
        assert (q_out[q_start[-1]:] == 7.0).all(), "rows behind the last sequence are left alone"
    for i, (name, want, mag, raw) in enumerate((("k", wk, mk, k64), ("v", v64, 0 * v64, v64))):
        pages = (B.cache.k_pages, B.cache.v_pages)[i]
        got = pages[page_of, :, slot].cpu()
        if fp8:
            limit = R.key_limit(m) if scaling and name == "k" else 448.0
            exp = (B.cache.k_exp, B.cache.v_exp)[i]
            e = np.array([[R.exponent(float(np.abs(raw[t, h]).max()), limit) for h in range(K)] for t in range(len(tok))])
            assert np.array_equal(exp[page_of, :, slot].cpu().numpy().astype(int), e + 127)
            s = 2.0 ** e[..., None]
            codes = got.view(torch.float8_e4m3fn).float().double().numpy()
            err = np.abs(codes * s - want)
            bound = R.ROPE_ERR * mag * 1.07 + np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * s)
            exp_before = exps[i].clone()
            exp_before[page_of, :, slot] = exp[page_of, :, slot]
            assert torch.equal(exp, exp_before), "exponents of other slots"
        else:
            err = np.abs(got.double().numpy() - want)
            bound = R.ROPE_ERR * mag + 2.0 ** -8 * np.abs(want) + 1e-38
        assert (err <= bound).all(), (name, (err / bound).max())
        before = pool[:, i].clone()
        before[page_of, :, slot] = pages[page_of, :, slot].view(before.dtype)
        assert torch.equal(pages.view(before.dtype), before), "other slots"
    # and back, as they stand
    for dtype in (torch.bfloat16, torch.float32):
        back = [torch.full((T, K, D), 3.0, dtype=dtype, device=DEV) for _ in range(2)]
        gpu.kv_read_paged(B.cache, B.q_start, B.kv_len, *back)
        for x, vals in zip(back, B.values()):
            assert torch.equal(x[tok].cpu().double(), vals[page_of, :, slot]), "codes and bf16 rows come back exactly"
            assert (x[q_start[-1]:] == 3.0).all()
    return B


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,cached,H,K,D,page,scaling,rot,interleaved", [
    ([1], [0], 1, 1, 128, 16, "none", 128, False),
    ([1, 1, 1, 1, 1], [15, 16, 0, 1000, 31], 32, 8, 128, 16, "by_parts", 128, False),
    ([5, 0, 1, 130], [0, 40, 63, 30], 6, 2, 128, 64, "ntk", 64, False),
    ([300], [128], 12, 4, 64, 128, "linear", 32, True),
    ([33, 64, 1], [0, 0, 7], 3, 3, 64, 32, None, 64, False),
    ([700, 1, 2], [3, 0, 90], 8, 1, 128, 32, "none", 128, True),
])
def test_append_and_read_back(gpu, fp8, src, new, cached, H, K, D, page, scaling, rot, interleaved):
    append_case(gpu, sum(new) + D, new, cached, H, K, D, page, fp8, src, scaling, rot, interleaved)


def test_append_large_steps_and_many_sequences(gpu):
    """More tokens than four a CTA, and more sequences than one round of the search covers."""
    append_case(gpu, 9, [1] * 100 + [0] * 20 + [37] * 20, [i % 50 for i in range(140)], 2, 2, 64, 16, True, torch.bfloat16,
                "none", 64, False)
    append_case(gpu, 10, [1500, 1], [0, 5], 2, 1, 128, 16, False, torch.bfloat16, "none", 128, False)


def test_append_without_q_start_is_one_token_each(gpu):
    K, D = 2, 128
    lens = [5, 17, 1]
    A, B = (Batch(3, [0, 1, 2, 3], lens, K, D, 16, True) for _ in range(2))
    k, v = (normal(s, 3, K, D).to(torch.bfloat16).to(DEV) for s in (1, 2))
    plan = gpu.rope_plan(128)
    gpu.kv_append_paged(A.cache, k, v, A.q_start, A.kv_len, rope=plan)
    gpu.kv_append_paged(B.cache, k, v, None, B.kv_len, rope=plan)
    assert torch.equal(A.pool, B.pool) and torch.equal(A.cache.k_exp, B.cache.k_exp)


def test_e4m3_rows_of_extreme_values(gpu):
    """Infinities and NaN become the NaN code and leave their row's other values alone; largest and smallest rows."""
    K, D, page = 1, 64, 16
    B = Batch(4, [0, 8], [8], K, D, page, True)
    v = normal(7, 8, K, D)
    v[0, 0, 3], v[1, 0, 5], v[2, 0, 0] = float("inf"), float("-inf"), float("nan")
    v[3] = 0.0
    v[4] *= 1e38
    v[5] *= 1e-38
    v[6] = 448.0 * 2.0 ** 3   # exactly at the border of a scale
    v[7] = float("inf")
    v = v.to(DEV)
    gpu.kv_append_paged(B.cache, v, v, B.q_start, B.kv_len)
    out = [torch.empty(8, K, D, dtype=torch.float32, device=DEV) for _ in range(2)]
    gpu.kv_read_paged(B.cache, B.q_start, B.kv_len, *out)
    for x in out:
        x, w = x.cpu().double(), v.cpu().double()
        assert torch.equal(torch.isnan(x), ~torch.isfinite(w))
        fine = torch.isfinite(w[:3])
        assert ((x[:3] - w[:3]).abs()[fine] <= 2.0 ** -4 * w[:3].abs()[fine] + 2.0 ** -10 * 2.0 ** -6).all()
        assert not x[3].any()
        assert ((x[4] - w[4]).abs() <= 2.0 ** -4 * w[4].abs() + 2.0 ** 110).all()
        assert (x[5].abs() <= 2.0 ** -100).all()
        assert torch.equal(x[6], w[6])


def test_bad_tables_and_lengths_touch_nothing(gpu):
    """Entries outside the pool and lengths out of range are recorded; what is in range still works."""
    K, D, page = 2, 128, 16
    for fp8 in (False, True):
        B = Batch(5, [0, 2, 4], [20, 20], K, D, page, fp8)
        k = torch.ones(4, K, D, dtype=torch.bfloat16, device=DEV)
        good = B.cache.block_table[1, 1].item()
        for bad in (-1, B.pages, 2 ** 31 - 1, -2 ** 31):
            B.cache.block_table[1, 1] = bad
            before = B.pool.clone()
            gpu.kv_append_paged(B.cache, k, k, B.q_start, B.kv_len)
            assert gpu.device_error() == ERR_KV_TABLE
            page0 = int(B.table_cpu[0, 1])
            before[page0] = B.pool[page0]
            assert torch.equal(before, B.pool)
            out = [torch.full((4, K, D), 9.0, dtype=torch.float32, device=DEV) for _ in range(2)]
            gpu.kv_read_paged(B.cache, B.q_start, B.kv_len, *out)
            assert gpu.device_error() == ERR_KV_TABLE
            assert not out[0][2:].any() and (out[0][:2] != 9.0).any()
            o = torch.full((4, 4, D), 9.0, dtype=torch.bfloat16, device=DEV)
            gpu.attention_paged(torch.ones(4, 4, D, dtype=torch.bfloat16, device=DEV), B.cache, o, B.q_start, B.kv_len, 2, 0.1)
            assert gpu.device_error() == ERR_KV_TABLE
            assert torch.isfinite(o.float()).all()
        B.cache.block_table[1, 1] = good
        for lens in ([20, 33], [20, 1], [20, -5], [20, 2 ** 31 - 1]):  # past the table; below the new tokens; negative
            before = B.pool.clone()
            gpu.kv_append_paged(B.cache, k, k, B.q_start, i32(lens))
            assert gpu.device_error() == ERR_KV_SEQ
            keep = [int(x) for x in set(B.table_cpu[0].tolist() + B.table_cpu[1].tolist())]
            others = [i for i in range(B.pages) if i not in keep]
            assert torch.equal(before[others], B.pool[others])


# ---- attention over pages -----------------------------------------------------------------


def paged_case(gpu, seed, new, cached, H, K, D, page, fp8, scale=None, behind=2, poison=True, workspace=None, strided=False):
    q_start = [0]
    for n in new:
        q_start.append(q_start[-1] + n)
    T = q_start[-1] + behind
    kv_len = [max(0, a + n) for a, n in zip(cached, new)]
    B = Batch(seed, q_start, kv_len, K, D, page, fp8)
    vals = B.values()
    if poison:
        B.poison_unused()
    q = normal(seed + 3, T, H + (1 if strided else 0), D, scale=1.3).to(torch.bfloat16).to(DEV)[:, :H]
    out = torch.full((T, H + (2 if strided else 0), D), 5.0, dtype=torch.bfloat16, device=DEV)[:, :H]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    max_q = max(new + [0])
    gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, max_q, scale, workspace=workspace)
    torch.cuda.synchronize()
    check_attention(B, vals, q, out, new, cached, scale, D)
    if behind:
        assert (out[q_start[-1]:] == 5.0).all(), "rows behind the last sequence are left alone"
    return B, q, out


def check_attention(B, vals, q, out, new, cached, scale, D):
    q_start = B.q_start_list
    for b, (n, a) in enumerate(zip(new, cached)):
        if n == 0:
            continue
        k, v = (R.gather(x, B.table_cpu, b, B.kv_len_list[b]) for x in vals)
        qq = q[q_start[b]:q_start[b] + n].cpu().double()
        want, mag, big = R.attend(qq, k, v, a, scale)
        err = (out[q_start[b]:q_start[b] + n].cpu().double() - want).abs()
        bound = R.attention_bound(want, mag, big, D)
        assert (err <= bound).all(), (b, float((err / bound).max()))
        empty = [i for i in range(n) if a + i + 1 <= 0]
        assert not out[[q_start[b] + i for i in empty]].any(), "a row that sees nothing gives zeros"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,K,D", [(32, 8, 128), (8, 8, 128), (4, 2, 128), (8, 1, 128), (16, 1, 128), (3, 1, 64), (12, 2, 64),
                                   (24, 2, 128), (7, 7, 64), (20, 1, 128), (64, 1, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_head_groups(gpu, fp8, H, K, D, page):
    """One new token a sequence: every grouping of heads, ragged contexts down to a single position."""
    cached = [0, 300, 15, 16, 129]
    paged_case(gpu, H + D + page, [1] * 5, cached, H, K, D, page, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("cached", [[0], [14], [15], [16], [127], [128], [4095], [1, 2000, 777]])
def test_decode_lengths(gpu, fp8, page, cached):
    paged_case(gpu, 11 + page + len(cached), [1] * len(cached), cached, 8, 2, 128, page, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached,H,K,D,page", [
    ([2], [0], 4, 1, 128, 16),
    ([4, 1, 3], [100, 0, 17], 8, 2, 128, 16),        # a few drafted tokens
    ([16, 9], [500, 1000], 32, 8, 128, 32),
    ([17], [0], 4, 4, 64, 16),
    ([64], [64], 8, 2, 128, 64),
    ([65], [63], 8, 2, 128, 64),
    ([130, 0, 1, 31], [3, 50, 127, 1], 8, 2, 128, 32),
    ([129], [255], 6, 2, 64, 16),                    # groups of three heads
    ([200], [0], 3, 3, 128, 16),                     # one head each
    ([100], [900], 12, 1, 128, 128),                 # twelve heads on one
    ([40, 260], [0, 0], 20, 1, 64, 64),              # twenty
    ([300], [1], 16, 2, 128, 64),
])
def test_chunks(gpu, fp8, new, cached, H, K, D, page):
    paged_case(gpu, sum(new) + H, new, cached, H, K, D, page, fp8, strided=True)


@pytest.mark.parametrize("fp8", [False, True])
def test_lengths_below_the_new_tokens_leave_rows_empty(gpu, fp8):
    """kv_len < n_b: the first rows see nothing and give zeros, the error word says so."""
    for new, cached in (([5], [-3]), ([40], [-40]), ([1, 1], [-1, 4]), ([200, 3], [-150, 0])):
        paged_case(gpu, 21, new, cached, 8, 2, 128, 16, fp8)
    gpu.device_error()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(gpu, fp8, scale):
    """Even weights, a negative scale, and scores of hundreds (one position takes it all)."""
    paged_case(gpu, 31, [1, 40], [130, 77], 8, 2, 128, 16, fp8, scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [[3], [1], [13], [70], [200]])
def test_values_behind_the_mask_never_reach_a_row(gpu, fp8, new):
    """NaN keys and infinite values at a later new token: earlier rows are finite and right, later ones follow the
    arithmetic (NaN)."""
    n = new[0]
    H, K, D, page, a = 8, 2, 128, 16, 37
    B = Batch(41, [0, n], [a + n], K, D, page, fp8)
    bad = a + n // 2  # the token that is not finite
    pg, slot = int(B.table_cpu[0, bad // page]), bad % page
    vals = [x.clone() for x in B.values()]
    B.cache.k_pages[pg, 0, slot, 5] = 0x7f if fp8 else float("nan")
    B.cache.v_pages[pg, 1, slot, 9] = 0x7f if fp8 else float("inf")
    q = normal(42, n, H, D).to(torch.bfloat16).to(DEV)
    out = torch.empty_like(q)
    gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, n, 0.1)
    o = out.cpu().double()
    k, v = (R.gather(x, B.table_cpu, 0, a + n) for x in vals)
    want, mag, big = R.attend(q.cpu().double(), k, v, a, 0.1)
    bound = R.attention_bound(want, mag, big, D)
    clean = n // 2  # rows before the bad token
    assert ((o[:clean] - want[:clean]).abs() <= bound[:clean]).all()
    rest = o[clean:]
    assert torch.isnan(rest[:, :4]).all(), "kv head 0: a NaN key's score"
    hit = rest[:, 4:, 9]
    assert (torch.isnan(hit) if fp8 else hit == float("inf")).all()
    others = [d for d in range(D) if d != 9]
    assert ((rest[:, 4:][..., others] - want[clean:, 4:][..., others]).abs() <= bound[clean:, 4:][..., others]).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,new,a", [(8, 3, 37), (8, 7, 0), (8, 7, 700), (8, 13, 5), (8, 70, 200), (16, 200, 60), (4, 1000, 100)])
def test_huge_values_behind_the_mask_never_reach_a_row(gpu, fp8, H, new, a):
    """Values near the top of the range at the later new tokens: the weights that earlier rows give them are exactly zero,
    and nothing of the earlier rows' own values is lost to their size."""
    K, D, page = 2, 128, 16
    B = Batch(45 + new, [0, new], [a + new], K, D, page, fp8)
    clean = new // 2
    vals = [x.clone() for x in B.values()]
    for j in range(a + clean, a + new):
        pg, slot = int(B.table_cpu[0, j // page]), j % page
        if fp8:
            B.cache.v_exp[pg, :, slot] = 240
        else:
            B.cache.v_pages[pg, :, slot] = 1e37
    q = normal(46, new, H, D).to(torch.bfloat16)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), B.cache, out, B.q_start, B.kv_len, new, 0.1)
    k, v = (R.gather(x, B.table_cpu, 0, a + new) for x in vals)
    want, mag, big = attend_on_gpu(q[:clean].double(), k[:a + clean], v[:a + clean], a, 0.1)
    err = (out[:clean].cpu().double() - want).abs()
    bound = R.attention_bound(want, mag, big, D)
    assert (err <= bound).all(), float((err / bound).max())


def test_infinite_scores_and_masked_extremes(gpu):
    """A largest-value key gives one position all the weight; every score at the type's lowest still averages."""
    K, D, page = 1, 128, 16
    B = Batch(51, [0, 1], [33], K, D, page, False)
    big = torch.finfo(torch.bfloat16).max
    B.cache.k_pages.fill_(-1.0)
    q = torch.full((1, 4, D), 1.0, dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(q)
    gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, 1, 1e30)  # every score is -1.28e32
    v = R.gather(B.values()[1], B.table_cpu, 0, 33)
    mean = v.mean(0)
    assert ((out[0].cpu().double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -8 * v.abs().mean(0)).all()
    pg, slot = int(B.table_cpu[0, 1]), 4
    B.cache.k_pages[pg, 0, slot] = big / 256
    gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, 1, 1e-3)
    assert torch.equal(out[0].cpu().double(), v[20].expand(4, D))


def test_long_cache_and_large_strides(gpu):
    """A context past 32,000 positions in a pool whose elements pass 2^31."""
    K, D, page = 2, 128, 64
    n_pages = 140_000  # 140,000 * 2 * 64 * 128 elements = 2.3e9
    pool = torch.empty((n_pages, K, page, D), dtype=torch.uint8, device=DEV)
    exp = torch.empty((n_pages, K, page), dtype=torch.uint8, device=DEV)
    length = 33_001
    need = -(-length // page)
    ids = torch.linspace(n_pages - 1, n_pages // 2, need).to(torch.int32)  # far pages, descending
    assert len(set(ids.tolist())) == need
    codes = (normal(61, need, K, page, D) * 60).to(torch.float8_e4m3fn).view(torch.uint8)
    e = torch.randint(120, 124, (need, K, page), dtype=torch.uint8)
    pool[ids.long().to(DEV)] = codes.to(DEV)
    exp[ids.long().to(DEV)] = e.to(DEV)
    cache = PagedKv(pool, pool, ids[None].contiguous().to(DEV), exp, exp)
    vals = R.values(codes, e).transpose(1, 2).flatten(0, 1)[:length]
    for n in (1, 40):
        q = normal(62, n, 8, D).to(torch.bfloat16).to(DEV)
        out = torch.empty_like(q)
        gpu.attention_paged(q, cache, out, i32([0, n]), i32([length]), n, 0.09)
        want, mag, big = R.attend(q.cpu().double(), vals, vals, length - n, 0.09)
        err = (out.cpu().double() - want).abs()
        assert (err <= R.attention_bound(want, mag, big, D)).all()


def test_many_sequences(gpu):
    """More sequences than SMs, lengths of every kind, empty ones between."""
    rng = np.random.default_rng(5)
    cached = [int(x) for x in rng.integers(0, 400, 200)]
    new = [1] * 200
    paged_case(gpu, 71, new, cached, 4, 2, 128, 16, True)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    paged_case(gpu, 72, new, cached, 4, 1, 64, 32, False)
    new[17] = 150
    paged_case(gpu, 73, new, cached, 4, 1, 64, 32, True)


def test_repeats_give_the_same_bits_on_one_workspace(gpu):
    ws = gpu.attention_paged_workspace(Batch(80, [0, 1], [4100], 2, 128, 16, False).cache, 8, 4000, 1000, 32)
    for new, cached in (([1] * 4, [4000, 3, 900, 0]), ([100, 3], [3000, 9]), ([600], [0])):
        B, q, out = paged_case(gpu, 81, new, cached, 8, 2, 128, 16, False, workspace=ws, behind=0)
        for _ in range(3):
            again = torch.empty_like(out)
            gpu.attention_paged(q, B.cache, again, B.q_start, B.kv_len, max(new), 1 / math.sqrt(128), workspace=ws)
            assert torch.equal(again, out)


def test_a_sequence_over_max_q_is_left_out_and_recorded(gpu):
    for new in ([1, 3, 1], [30, 60, 2]):
        q_start = [0, new[0], new[0] + new[1], sum(new)]
        B = Batch(91, q_start, [50, 60, 70], 2, 128, 16, False)
        q = normal(92, sum(new), 8, 128).to(torch.bfloat16).to(DEV)
        out = torch.full_like(q, 5.0)
        gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, max(new[0], new[2]), 0.1)
        torch.cuda.synchronize()
        assert gpu.device_error() == ERR_KV_SEQ
        assert (out[q_start[1]:q_start[2]] == 5.0).all()
        assert not (out[:q_start[1]] == 5.0).all() and not (out[q_start[2]:] == 5.0).all()


def test_a_workspace_serves_smaller_batches(gpu):
    """A cache so wide that the bf16 copy of two sequences' codes is past its limit, and that of one is not."""
    K, D, page, width, a, n = 8, 128, 64, 2100, 900, 200
    B = Batch(85, [0, n], [a + n], K, D, page, True)
    table = torch.zeros((2, width), dtype=torch.int32, device=DEV)
    table[:1, :B.cache.block_table.shape[1]] = B.cache.block_table
    B.cache = PagedKv(B.cache.k_pages, B.cache.v_pages, table, B.cache.k_exp, B.cache.v_exp)
    q = normal(86, n, 32, D).to(torch.bfloat16).to(DEV)
    ws = gpu.attention_paged_workspace(B.cache, 2, 2 * n, n, 32)
    for workspace in (ws, None):
        out = torch.empty_like(q)
        gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, n, 0.1, workspace=workspace)
        check_attention(B, B.values(), q, out, [n], [a], 0.1, D)


def test_attention_refuses(gpu):
    B = Batch(95, [0, 1], [5], 2, 128, 16, False)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(q)
    with pytest.raises(TypeError):
        gpu.attention_paged(q.float(), B.cache, out, B.q_start, B.kv_len, 1, 0.1)
    with pytest.raises(TypeError):
        gpu.attention_paged(q, B.cache, out.float(), B.q_start, B.kv_len, 1, 0.1)
    with pytest.raises(ValueError):
        gpu.attention_paged(q[..., :64], B.cache, out[..., :64], B.q_start, B.kv_len, 1, 0.1)
    with pytest.raises(ValueError):
        gpu.attention_paged(q, B.cache, out, B.q_start.cpu(), B.kv_len, 1, 0.1)
    with pytest.raises(ValueError):
        gpu.attention_paged(q, B.cache, out, i32([0, 1, 1]), B.kv_len, 1, 0.1)
    with pytest.raises(ValueError):
        gpu.attention_paged(q, B.cache, out, i32([0, 1, 1, 1]), i32([5, 5, 5]), 1, 0.1)  # more sequences than table rows
    with pytest.raises(Exception):
        gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, 1, 0.1, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(Exception):
        gpu.attention_paged(q[:, :7], B.cache, out[:, :7], B.q_start, B.kv_len, 1, 0.1)
    with pytest.raises(Exception):
        gpu.attention_paged(q, B.cache, q, B.q_start, B.kv_len, 1, 0.1)  # rows are read again after others are written


def attend_on_gpu(q, k, v, n_before, scale):
    """R.attend for larger cases: float64 matrices on the GPU, a head at a time."""
    n, H, D = q.shape
    L, K, _ = k.shape
    q, k, v = (x.to(DEV).double() for x in (q, k, v))
    later = torch.arange(L, device=DEV)[None] > torch.arange(n_before, n_before + n, device=DEV)[:, None]
    out, mag, big = (torch.empty(n, H, d, dtype=torch.float64, device=DEV) for d in (D, D, 1))
    for h in range(H):
        kk, vv = k[:, h // (H // K)], v[:, h // (H // K)]
        p = (q[:, h] @ kk.T * scale).masked_fill(later, float("-inf")).softmax(-1)
        out[:, h], mag[:, h] = p @ vv, p @ vv.abs()
        big[:, h, 0] = (q[:, h].abs() @ kk.abs().T).masked_fill(later, 0.0).amax(-1) * abs(scale)
    return out.cpu(), mag.cpu(), big.cpu()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,cached,H,K,D,page", [
    ([40], [20001], 8, 2, 128, 64),              # a long cache split over the SMs
    ([700, 33], [5000, 2500], 8, 2, 128, 32),    # chunks of several tiles beside a short one
    ([3, 1, 2], [15000, 60, 9000], 16, 1, 64, 16),
    ([1500], [0], 4, 1, 64, 128),
])
def test_larger_chunks(gpu, fp8, new, cached, H, K, D, page):
    q_start = [0]
    for n in new:
        q_start.append(q_start[-1] + n)
    B = Batch(300 + sum(new), q_start, [a + n for a, n in zip(cached, new)], K, D, page, fp8)
    vals = B.values()
    B.poison_unused()
    q = normal(301, q_start[-1], H, D, scale=1.3).to(torch.bfloat16)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), B.cache, out, B.q_start, B.kv_len, max(new), 1 / math.sqrt(D))
    for b, (n, a) in enumerate(zip(new, cached)):
        k, v = (R.gather(x, B.table_cpu, b, a + n) for x in vals)
        s = slice(q_start[b], q_start[b + 1])
        want, mag, big = attend_on_gpu(q[s], k, v, a, 1 / math.sqrt(D))
        err = (out[s].cpu().double() - want).abs()
        bound = R.attention_bound(want, mag, big, D)
        assert (err <= bound).all(), (b, float((err / bound).max()))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [1, 3, 30, 200])
def test_scores_that_keep_rising(gpu, fp8, new):
    """Every tile passes the running maximum by far: the outputs so far are scaled down again and again."""
    H, K, D, page, a = 8, 2, 128, 32, 900
    B = Batch(310, [0, new], [a + new], K, D, page, fp8)
    g = normal(311, D)
    for j in range(a + new):  # keys along one direction, longer and longer
        row = (g * (0.02 + j / 300.0))
        pg, slot = int(B.table_cpu[0, j // page]), j % page
        if fp8:
            e = R.exponent(float(row.abs().max()), 448.0)
            B.cache.k_pages[pg, :, slot] = (row * 2.0 ** -e).to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
            B.cache.k_exp[pg, :, slot] = e + 127
        else:
            B.cache.k_pages[pg, :, slot] = row.to(torch.bfloat16).to(DEV)
    vals = B.values()
    q = (g + normal(312, new, H, D, scale=0.3)).to(torch.bfloat16)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=DEV)
    gpu.attention_paged(q.to(DEV), B.cache, out, B.q_start, B.kv_len, new, 0.3)
    k, v = (R.gather(x, B.table_cpu, 0, a + new) for x in vals)
    want, mag, big = R.attend(q.double(), k, v, a, 0.3)
    err = (out.cpu().double() - want).abs()
    assert (err <= R.attention_bound(want, mag, big, D)).all()


@pytest.mark.parametrize("new", [1, 3, 30, 200])
@pytest.mark.parametrize("rising", [False, True])
def test_rows_of_very_unlike_exponents(gpu, new, rising):
    """e4m3 rows whose powers of two span 2^24, in no order and growing along the sequence."""
    H, K, D, page, a = 8, 2, 128, 16, 700
    B = Batch(320, [0, new], [a + new], K, D, page, True)
    gen = torch.Generator().manual_seed(5)
    for j in range(a + new):
        pg, slot = int(B.table_cpu[0, j // page]), j % page
        for exp in (B.cache.k_exp, B.cache.v_exp):
            e = 110 + 24 * j // (a + new) if rising else int(torch.randint(110, 134, (1,), generator=gen))
            exp[pg, :, slot] = e
    vals = B.values()
    q = normal(321, new, H, D).to(torch.bfloat16)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=DEV)
    scale = 1e-4
    gpu.attention_paged(q.to(DEV), B.cache, out, B.q_start, B.kv_len, new, scale)
    k, v = (R.gather(x, B.table_cpu, 0, a + new) for x in vals)
    want, mag, big = R.attend(q.double(), k, v, a, scale)
    err = (out.cpu().double() - want).abs()
    bound = R.attention_bound(want, mag, big, D)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [[1] * 1100, [1, 0, 2] * 400, [40] + [1] * 1100])
def test_more_sequences_than_any_list_holds(gpu, fp8, new):
    cached = [(7 * i) % 45 for i in range(len(new))]
    paged_case(gpu, 330, new, cached, 2, 1, 64, 16, fp8)


def test_sequences_that_share_pages(gpu):
    """Two sequences with a common prefix: the same pages in both rows of the table."""
    K, D, page = 2, 128, 16
    B = Batch(340, [0, 1, 41], [100, 140], K, D, page, False)
    B.table_cpu[1, :6] = B.table_cpu[0, :6]
    B.cache.block_table.copy_(B.table_cpu)
    vals = B.values()
    q = normal(341, 41, 8, D).to(torch.bfloat16).to(DEV)
    out = torch.empty_like(q)
    gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, 40, 0.1)
    check_attention(B, vals, q, out, [1, 40], [99, 100], 0.1, D)


def test_wide_and_strided_tables(gpu):
    """A block table cut out of a wider one, its unused entries out of range: never read past a sequence's length."""
    K, D, page = 2, 128, 16
    B = Batch(350, [0, 1, 2], [100, 33], K, D, page, True)
    vals = B.values()
    wide = torch.full((2, 50), -7, dtype=torch.int32)
    for b, n in enumerate((7, 3)):
        wide[b, 5:5 + n] = B.table_cpu[b, :n]
    cache = PagedKv(B.cache.k_pages, B.cache.v_pages, wide.to(DEV)[:, 5:45], B.cache.k_exp, B.cache.v_exp)
    for n in (1, 30):
        q_start = [0, 1, 1 + n]
        lens = [100, 33]
        q = normal(351, 1 + n, 8, D).to(torch.bfloat16).to(DEV)
        out = torch.empty_like(q)
        gpu.attention_paged(q, cache, out, i32(q_start), i32(lens), n, 0.1)
        B.q_start_list, B.kv_len_list = q_start, lens
        check_attention(B, vals, q, out, [1, n], [99, 33 - n], 0.1, D)


# ---- attention over prompts ----------------------------------------------------------------


def prompt_case(gpu, seed, new, H, K, D, behind=2, fused=True, scale=None):
    q_start = [0]
    for n in new:
        q_start.append(q_start[-1] + n)
    T = q_start[-1] + behind
    rows = normal(seed, T, (H + 2 * K) * D, scale=1.2).to(torch.bfloat16)
    rows[q_start[-1]:] = float("nan")  # what lies behind the last sequence is nobody's
    rows = rows.to(DEV)
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    out = torch.full((T, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    gpu.attention_prompt(q, k, v, out, i32(q_start), max(new), scale)
    torch.cuda.synchronize()
    for b, n in enumerate(new):
        if n == 0:
            continue
        s = slice(q_start[b], q_start[b + 1])
        want, mag, big = R.attend(q[s].cpu().double(), k[s].cpu().double(), v[s].cpu().double(), 0, scale)
        err = (out[s].cpu().double() - want).abs()
        bound = R.attention_bound(want, mag, big, D)
        assert (err <= bound).all(), (b, float((err / bound).max()))
    assert (out[q_start[-1]:] == 5.0).all()


@pytest.mark.parametrize("new,H,K,D", [
    ([1], 1, 1, 128), ([1], 32, 8, 128), ([2, 1, 1], 4, 4, 64), ([31, 33], 8, 2, 128), ([63, 0, 65], 8, 2, 128),
    ([127, 1, 128], 4, 1, 128), ([129], 6, 2, 64), ([256], 3, 1, 128), ([255, 257], 5, 5, 128), ([500, 3], 16, 1, 128),
    ([300, 301], 20, 1, 64), ([1030], 8, 2, 128), ([64] * 9, 2, 2, 64)])
@pytest.mark.parametrize("fused", [False, True])
def test_prompts(gpu, new, H, K, D, fused):
    prompt_case(gpu, sum(new) + H, new, H, K, D, fused=fused)


def test_prompt_neighbours_never_mix(gpu):
    """A prompt full of NaN beside two others."""
    H, K, D = 8, 2, 128
    new = [70, 90, 40]
    rows = normal(5, 200, (H + 2 * K) * D).to(torch.bfloat16).to(DEV)
    clean = torch.empty(200, H, D, dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(clean)
    split = lambda r: [r[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K))]  # noqa: E731
    gpu.attention_prompt(*split(rows), clean, i32([0, 70, 160, 200]), 90, 0.1)
    bad = rows.clone()
    bad[70:160] = float("nan")
    gpu.attention_prompt(*split(bad), out, i32([0, 70, 160, 200]), 90, 0.1)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[160:], clean[160:])
    assert torch.isnan(out[70:160]).all()


def test_huge_values_behind_the_mask_of_a_prompt(gpu):
    H, K, D, n = 8, 2, 128, 300
    q, k, v = (normal(6 + i, n, h, D).to(torch.bfloat16) for i, h in enumerate((H, K, K)))
    v[100:] = 1e37
    out = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
    gpu.attention_prompt(q.to(DEV), k.to(DEV), v.to(DEV), out, i32([0, n]), n, 0.1)
    want, mag, big = R.attend(q[:100].double(), k[:100].double(), v[:100].double(), 0, 0.1)
    err = (out[:100].cpu().double() - want).abs()
    bound = R.attention_bound(want, mag, big, D)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("new,H,K,D", [([3000, 1501], 4, 1, 128), ([2200], 3, 3, 64), ([700] * 5, 12, 2, 128)])
def test_larger_prompts(gpu, new, H, K, D):
    q_start = [0]
    for n in new:
        q_start.append(q_start[-1] + n)
    rows = normal(400, q_start[-1], (H + 2 * K) * D).to(torch.bfloat16).to(DEV)
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=DEV)
    gpu.attention_prompt(q, k, v, out, i32(q_start), max(new), 0.1)
    for b in range(len(new)):
        s = slice(q_start[b], q_start[b + 1])
        want, mag, big = attend_on_gpu(q[s], k[s], v[s], 0, 0.1)
        err = (out[s].cpu().double() - want).abs()
        assert (err <= R.attention_bound(want, mag, big, D)).all()


# ---- together ------------------------------------------------------------------------------


def test_a_prompt_and_its_decode_steps(gpu):
    """rotate + append + attend in chunks and single tokens gives what the prompt attention gives at once."""
    H, K, D, page, n = 8, 2, 128, 16, 150
    plan = gpu.rope_plan(128)
    rows = normal(7, n, (H + 2 * K) * D).to(torch.bfloat16).to(DEV)
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    whole = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
    gpu.attention_prompt(gpu.rope(q, pos, plan), gpu.rope(k, pos, plan), v, whole, i32([0, n]), n, 0.09)
    for fp8 in (False, True):
        table = torch.randperm(12).to(torch.int32)[None, :10].to(DEV)
        cache = PagedKv.empty(12, K, page, D, table, fp8=fp8)
        out, at = torch.empty_like(whole), 0
        for step in (100, 1, 1, 30, 5, 1, 12):
            s = slice(at, at + step)
            q_rot = torch.empty(step, H, D, dtype=torch.bfloat16, device=DEV)
            gpu.kv_append_paged(cache, k[s], v[s], i32([0, step]), i32([at + step]), rope=plan, q=q[s], q_out=q_rot)
            gpu.attention_paged(q_rot, cache, out[s], i32([0, step]), i32([at + step]), step, 0.09)
            at += step
        kr, vr = (torch.empty(n, K, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        gpu.kv_read_paged(cache, i32([0, n]), i32([n]), kr, vr)
        q_rot = gpu.rope(q, pos, plan)
        want, mag, big = R.attend(q_rot.cpu().double(), kr.cpu().double(), vr.cpu().double(), 0, 0.09)
        bound = R.attention_bound(want, mag, big, D)
        assert ((out.cpu().double() - want).abs() <= bound).all()
        if not fp8:
            assert torch.equal(kr, gpu.rope(k, pos, plan)) and torch.equal(vr, v)
            assert ((whole.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 1]])
def test_captured_steps_replay_with_new_lengths(gpu, new):
    """A captured append + attention replayed as the sequences grow: lengths and tables are read on the device."""
    H, K, D, page = 8, 2, 128, 16
    plan = gpu.rope_plan(128)
    T, q_start = sum(new), [0, new[0], new[0] + new[1], sum(new)]
    cached = [5, 100, 0]
    B = Batch(13, q_start, [a + 4 * n for a, n in zip(cached, new)], K, D, page, True)
    qkv = torch.zeros(T, (H + 2 * K) * D, dtype=torch.bfloat16, device=DEV)
    q, k, v = (qkv[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    q_rot, out = (torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lens = i32(cached)

    def step():
        lens.add_(i32_new)
        gpu.kv_append_paged(B.cache, k, v, B.q_start, lens, rope=plan, q=q, q_out=q_rot)
        gpu.attention_paged(q_rot, B.cache, out, B.q_start, lens, max(new), 0.09)

    i32_new = i32(new)
    pool = B.pool.clone()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    lens.copy_(i32(cached))
    B.pool.copy_(pool)
    got = []
    for i in range(4):
        qkv.copy_(normal(100 + i, T, (H + 2 * K) * D).to(torch.bfloat16))
        graphs[i % 2].replay()
        got.append(out.clone())
    lens.copy_(i32(cached))
    B.pool.copy_(pool)
    for i in range(4):
        qkv.copy_(normal(100 + i, T, (H + 2 * K) * D).to(torch.bfloat16))
        step()
        assert torch.equal(out, got[i]), i


def test_two_streams_at_once(gpu):
    """Calls on two streams keep apart (a workspace each), and order by their own stream."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i, (new, cached) in enumerate((([1, 1], [3000, 200]), ([90], [700]))):
        q_start = [0]
        for n in new:
            q_start.append(q_start[-1] + n)
        B = Batch(200 + i, q_start, [a + n for a, n in zip(cached, new)], 2, 128, 16, False)
        q = normal(210 + i, sum(new), 8, 128).to(torch.bfloat16).to(DEV)
        want = torch.empty_like(q)
        gpu.attention_paged(q, B.cache, want, B.q_start, B.kv_len, max(new), 0.1)
        cases.append((B, q, max(new), want))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (B, q, m, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                o = torch.zeros_like(q)
                gpu.attention_paged(q, B.cache, o, B.q_start, B.kv_len, m, 0.1)
                outs[i].append(o)
    torch.cuda.synchronize()
    for i, (_, _, _, want) in enumerate(cases):
        assert all(torch.equal(o, want) for o in outs[i])


def test_two_graphs_at_once(gpu):
    """Graphs captured from calls without a workspace have their own, so they may replay at the same time."""
    made = []
    for i, (new, cached) in enumerate((([1, 1, 1], [4000, 90, 2000]), ([120, 3], [900, 2000]))):
        q_start = [0]
        for n in new:
            q_start.append(q_start[-1] + n)
        B = Batch(500 + i, q_start, [a + n for a, n in zip(cached, new)], 2, 128, 16, True)
        q = normal(510 + i, sum(new), 8, 128).to(torch.bfloat16).to(DEV)
        want, out = torch.empty_like(q), torch.zeros_like(q)
        gpu.attention_paged(q, B.cache, want, B.q_start, B.kv_len, max(new), 0.1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(10):
                gpu.attention_paged(q, B.cache, out, B.q_start, B.kv_len, max(new), 0.1)
        made.append((g, B, q, want, out, torch.cuda.Stream()))
    for _ in range(5):
        for g, _, _, _, out, stream in made:
            with torch.cuda.stream(stream):
                out.zero_()
                g.replay()
        torch.cuda.synchronize()
        for _, _, _, want, out, _ in made:
            assert torch.equal(out, want)
