"""Timed cases of the paged key/value cache and of the prompt attention beside it.

Five operators of a serving step, each in a plain form (elementary torch
operations in fp32, angles in fp64, one rounding at the end) and as the calls a
user makes of `homelab_b200` (`own`):

  rope          rotary positions on [tokens, heads, head_dim] rows
  append        a step's keys and values (and its queries) rotated, written into a
                paged cache in bf16 or in e4m3 with one power-of-two scale per row
  read          cached positions back as contiguous rows
  paged         attention of each sequence's new tokens over its pages, causal
  prompt        causal attention over packed whole prompts

Sequences are packed: `new` and `cached` list every sequence's new tokens and the
positions cached before them.
"""
import functools
import math

import torch

own = False

DEV = "cuda"

# rotary settings a case names: (base, scaling, factor, original length)
ROPE = {
    "plain": (10000.0, "none", 1.0, 0),
    "linear": (10000.0, "linear", 4.0, 0),
    "ntk": (10000.0, "ntk", 8.0, 0),
    "by_parts": (500000.0, "by_parts", 16.0, 8192),
}


def _ints(text):
    return [int(v) for v in str(text).split(",")]


def _case(name, op, new, cached, heads, kv_heads, head_dim=128, cache="bf16", page=16, rope="plain", rot=None,
          interleaved=False, src="bf16"):
    c = {"op": op, "new": new, "cached": cached, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "cache": cache, "page": page, "rope": rope, "rot": rot or head_dim, "interleaved": interleaved, "src": src}
    if name:
        c["name"] = name
    return c


def listed():
    one = lambda n: ",".join(["1"] * n)  # noqa: E731
    return [
        # rotary positions of a decode batch's queries: 8 sequences, a launch-latency call
        _case("rope_decode", "rope", one(8), "4095,17,900,2047,3000,1,512,4000", 32, 8),
        # the queries of a long packed prompt; interleaved pairs over half of the head, context
        # stretched 16 times, fp32 rows out of an fp32 projection
        _case("rope_prompt_long", "rope", "8191,1200", "122880,0", 32, 8, rope="by_parts", rot=64, interleaved=True,
              src="f32"),
        # a decode step's write into an 8-bit cache: 32 sequences, one token each
        _case("append_decode_e4m3", "append", one(32), ",".join(str(127 * i) for i in range(32)), 32, 8,
              cache="e4m3"),
        # a prefill step's write: ragged chunks of four prompts into a bf16 cache
        _case("append_chunks_bf16", "append", "4096,1031,2500,565", "0,4096,77,12000", 32, 8, page=64, rope="ntk"),
        # one sequence's 8-bit pages read back (to move it to another pool or to host memory)
        _case("read_sequence_e4m3", "read", "2047", "0", 32, 8, cache="e4m3"),
        # a batch of long bf16 sequences read back
        _case("read_batch_bf16", "read", "16384,9001,12000,5000", "0,40,0,7", 32, 8, page=64),
        # single-sequence decode at 32 query heads over 8 kv heads, context 4096: latency
        _case("paged_decode_one", "paged", "1", "4095", 32, 8),
        # batched decode over 8-bit pages, ragged contexts
        _case("paged_decode_batch_e4m3", "paged", one(32), ",".join(str(1000 + 487 * i) for i in range(32)), 32, 8,
              cache="e4m3", page=64),
        # a few drafted tokens to verify, three sequences
        _case("paged_draft", "paged", "9,4,16", "8000,313,5000", 32, 4, page=32),
        # chunked prefill over a long 8-bit cache beside another sequence's chunk
        _case("paged_chunk_e4m3", "paged", "1024,512", "15360,4001", 32, 8, cache="e4m3", page=64),
        # a handful of short prompts, one token to a few hundred
        _case("prompt_short", "prompt", "1,37,300,128,5", "0,0,0,0,0", 32, 8),
        # two long prompts packed
        _case("prompt_long", "prompt", "8192,3001", "0,0", 32, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "paged", "paged", "prompt"])
    head_dim = rng.choice([128, 128, 64])
    group = rng.choice([1, 2, 3, 4, 4, 6, 8])
    kv_heads = rng.choice([1, 2, 4, 8]) if group > 1 else rng.choice([4, 8, 16])
    heads = group * kv_heads
    cache = rng.choice(["bf16", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    more = dict(head_dim=head_dim, cache=cache, page=page, rope=rng.choice(sorted(ROPE)),
                rot=rng.choice([head_dim, head_dim, head_dim // 2]), interleaved=rng.random() < 0.4,
                src=rng.choice(["bf16", "bf16", "f32"]) if op in ("rope", "append") else "bf16")
    batch = _log(rng, 1, 32)
    if op == "prompt":
        batch = _log(rng, 1, 8)
        new = [_log(rng, 1, 6000 / batch) for _ in range(batch)]
        cached = [0] * batch
    elif op == "paged":
        if rng.random() < 0.5:
            new = [1] * batch
            cached = [_log(rng, 1, 16000) - 1 for _ in range(batch)]
        else:
            batch = _log(rng, 1, 6)
            new = [_log(rng, 1, 1000 / batch) for _ in range(batch)]
            cached = [_log(rng, 1, 12000) - 1 for _ in range(batch)]
    elif op == "read":
        batch = _log(rng, 1, 8)
        new = [_log(rng, 1, 32000 / batch) for _ in range(batch)]
        cached = [rng.randrange(0, 200) for _ in range(batch)]
    else:
        new = [1] * batch if rng.random() < 0.4 else [_log(rng, 1, 6000 / batch) for _ in range(batch)]
        cached = [_log(rng, 1, 20000) - 1 for _ in range(batch)]
    return _case(None, op, ",".join(map(str, new)), ",".join(map(str, cached)), heads, kv_heads, **more)


# ---- inputs ------------------------------------------------------------------------------


def _quantise(x, limit):
    """e4m3 codes of rows x (fp32) under 2^e, e the least with amax <= limit * 2^e, and e + 127 as a byte."""
    amax = x.abs().amax(-1)
    e = _exponent(amax, limit)
    codes = (x * torch.exp2(-e.float())[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _exponent(amax, limit):
    m, e = torch.frexp(amax)
    ml, el = math.frexp(limit)
    return torch.where(amax > 0, e - el + (m > ml).int(), torch.zeros_like(e)).clamp(-100, 120)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, cached = _ints(c["new"]), _ints(c["cached"])
    B, T = len(new), sum(new)
    H, K, D, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    src = torch.float32 if c["src"] == "f32" else torch.bfloat16

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV) * scale

    s = {"case": dict(c), "max_q": max(new), "scale": 1.0 / math.sqrt(D)}
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    s["q_start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
    s["kv_len"] = torch.tensor([a + n for a, n in zip(cached, new)], dtype=torch.int32, device=DEV)
    if c["op"] == "rope":
        s["x"] = normal(T, H, D).to(src)
        s["positions"] = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(cached, new)]).to(DEV)
        return s
    # channels of unlike size, as keys have
    spread = torch.exp(normal(K, D, scale=0.4))
    if c["op"] in ("append", "prompt"):
        # the rows of one fused projection: queries, keys and values of a token side by side
        rows = normal(T, (H + 2 * K) * D)
        rows[:, H * D:(H + K) * D] *= spread.reshape(-1)
        rows = rows.to(src)
        s["q"] = rows[:, :H * D].unflatten(1, (H, D))
        s["k"] = rows[:, H * D:(H + K) * D].unflatten(1, (K, D))
        s["v"] = rows[:, (H + K) * D:].unflatten(1, (K, D))
        if c["op"] == "prompt":
            return s
    if c["op"] == "paged":
        s["q"] = normal(T, H, D).to(torch.bfloat16)
    need = [-(-(a + n) // ps) for a, n in zip(cached, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((B, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table
    for name in ("k", "v"):
        x = normal(pages, K, ps, D)
        if name == "k":
            x *= spread[:, None, :]
        if c["cache"] == "e4m3":
            s[name + "_pages"], s[name + "_exp"] = _quantise(x, 448.0)
        else:
            s[name + "_pages"] = x.to(torch.bfloat16)
    return s


# ---- the plain forms ---------------------------------------------------------------------


def _inv_freq(case):
    """Angle per position of each pair, fp64, and the factor on cos and sin."""
    base, scaling, factor, original = ROPE[case["rope"]]
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    inv = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "by_parts":
        # pairs turning more than 32 times over the original length keep their angle, those
        # turning less than once are stretched, a ramp between
        dim = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _rotate(x, positions, case):
    inv, m = _inv_freq(case)
    angle = positions.double()[:, None] * inv
    cos, sin = (angle.cos() * m).to(x.dtype)[:, None], (angle.sin() * m).to(x.dtype)[:, None]
    rot = case["rot"]
    r = x[..., :rot]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _places(s):
    """Sequence and cache position of every packed new token."""
    t = torch.arange(sum(_ints(s["case"]["new"])), device=DEV)
    seq = torch.searchsorted(s["q_start"][1:], t, right=True)
    return seq, t - s["q_start"][seq] + s["kv_len"][seq] - (s["q_start"][seq + 1] - s["q_start"][seq])


def _values(s, name, dtype=torch.float32):
    """The cache's rows as the values they stand for."""
    x = s[name + "_pages"].to(dtype)
    return x * torch.exp2(s[name + "_exp"].to(dtype) - 127)[..., None] if name + "_exp" in s else x


def _limit(case):
    """The largest input whose row, rotated, stays within +-448 under scale 1, rounded down to fp32."""
    m = _inv_freq(case)[1]
    limit = torch.tensor(448.0 / (math.sqrt(2.0) * m), dtype=torch.float64)
    f = limit.float()
    return float(torch.nextafter(f, torch.zeros_like(f)) if f.double() > limit else f)


def _plain_append(s):
    c = s["case"]
    seq, pos = _places(s)
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    q = _rotate(s["q"].float(), pos, c).to(torch.bfloat16)
    k, v = _rotate(s["k"].float(), pos, c), s["v"].float()
    if c["cache"] == "bf16":
        s["k_pages"][page, :, slot] = k.to(torch.bfloat16)
        s["v_pages"][page, :, slot] = v.to(torch.bfloat16)
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    for name, x, e in (("k", k, _exponent(s["k"].float().abs().amax(-1), _limit(c))),
                       ("v", v, _exponent(v.abs().amax(-1), 448.0))):
        codes = (x * torch.exp2(-e.float())[..., None]).to(torch.float8_e4m3fn)
        s[name + "_pages"].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
        s[name + "_exp"][page, :, slot] = (e + 127).to(torch.uint8)
    return {"q": q, "k": s["k_pages"], "v": s["v_pages"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _plain_read(s):
    c = s["case"]
    seq, pos = _places(s)
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    got = []
    for name in ("k", "v"):
        x = s[name + "_pages"].view(torch.uint8 if c["cache"] == "e4m3" else torch.bfloat16)[page, :, slot]
        if c["cache"] == "e4m3":
            x = x.view(torch.float8_e4m3fn).float() * torch.exp2(s[name + "_exp"][page, :, slot].float() - 127)[..., None]
        got.append(x.to(torch.bfloat16))
    return got


def _attend(q, k, v, q_start, kv_len, n_max, scale):
    """q [T, H, D] packed; k, v [B, L, K, D] padded; every new token sees the positions up to its own."""
    B, L, K, D = k.shape
    T, H, _ = q.shape
    n = (q_start[1:] - q_start[:-1])[:, None]
    i = torch.arange(n_max, device=DEV)[None]
    row = (q_start[:-1, None] + i).clamp(max=T - 1).long()
    qp = q[row].float().unflatten(2, (K, H // K))                                   # [B, n, K, G, D]
    qp = qp.permute(0, 2, 3, 1, 4).reshape(B, K, -1, D)                             # [B, K, G * n, D]
    s = (qp @ k.float().permute(0, 2, 3, 1)).mul_(scale).view(B, K, H // K, n_max, L)
    see = torch.arange(L, device=DEV)[None, None] <= (kv_len[:, None] - n + i)[..., None]
    s.masked_fill_(~see[:, None, None], float("-inf"))
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    out = (p.view(B, K, -1, L) @ v.float().permute(0, 2, 1, 3)).view(B, K, H // K, n_max, D)
    out = out / p.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n_max, H, D)
    return out[(i < n).expand(B, n_max)].to(torch.bfloat16)


def _plain_paged(s):
    c = s["case"]
    L = s["table"].shape[1] * c["page"]
    j = torch.arange(L, device=DEV)
    seen = (j[None] < s["kv_len"][:, None])[:, :, None, None]
    t = s["table"].long()
    k, v = (torch.where(seen, x, 0.0) for x in (_values_of(s, name, t) for name in ("k", "v")))
    return _attend(s["q"], k, v, s["q_start"], s["kv_len"], s["max_q"], s["scale"])


def _values_of(s, name, table):
    """[B, L, K, D]: the pages of every row of the table in order, fp32."""
    x = s[name + "_pages"]
    x = (x.view(torch.uint8)[table].view(torch.float8_e4m3fn) if x.dtype == torch.float8_e4m3fn else x[table]).float()
    if name + "_exp" in s:
        x = x * torch.exp2(s[name + "_exp"][table].float() - 127)[..., None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_prompt(s):
    n = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(s["max_q"], device=DEV)[None]
    row = (s["q_start"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    return _attend(s["q"], s["k"][row], s["v"][row], s["q_start"], n, s["max_q"], s["scale"])


# ---- the framework's calls ---------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _gpu():
    from homelab_b200.backend import Gpu
    return Gpu(torch.cuda.current_device())


@functools.lru_cache(maxsize=None)
def _rope(name, rot, interleaved):
    base, scaling, factor, original = ROPE[name]
    return _gpu().rope_plan(rot, base=base, scaling=scaling, factor=factor, original_len=original,
                            interleaved=interleaved)


def _own(s):
    c, gpu = s["case"], _gpu()
    rope = _rope(c["rope"], c["rot"], c["interleaved"])
    if c["op"] == "rope":
        out = torch.empty_like(s["x"])
        gpu.rope(s["x"], s["positions"], rope, out)
        return out
    if c["op"] == "prompt":
        out = torch.empty(s["q"].shape, dtype=torch.bfloat16, device=DEV)
        gpu.attention_prompt(s["q"], s["k"], s["v"], out, s["q_start"], s["max_q"], s["scale"])
        return out
    from homelab_b200.paged import PagedKv
    cache = PagedKv(s["k_pages"], s["v_pages"], s["table"], s.get("k_exp"), s.get("v_exp"))
    if c["op"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.bfloat16, device=DEV)
        gpu.kv_append_paged(cache, s["k"], s["v"], s["q_start"], s["kv_len"], rope=rope, q=s["q"], q_out=q)
        out = {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
        return out if c["cache"] == "bf16" else {**out, "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    if c["op"] == "read":
        T = sum(_ints(c["new"]))
        out = [torch.empty((T, c["kv_heads"], c["head_dim"]), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        gpu.kv_read_paged(cache, s["q_start"], s["kv_len"], out[0], out[1])
        return out
    out = torch.empty_like(s["q"])
    gpu.attention_paged(s["q"], cache, out, s["q_start"], s["kv_len"], s["max_q"], s["scale"])
    return out


PLAIN = {"rope": lambda s: _rotate(s["x"].float(), s["positions"], s["case"]).to(s["x"].dtype),
         "append": _plain_append, "read": _plain_read, "paged": _plain_paged, "prompt": _plain_prompt}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    c = case
    new, cached = _ints(c["new"]), _ints(c["cached"])
    B, T = len(new), sum(new)
    H, K, D = c["heads"], c["kv_heads"], c["head_dim"]
    src = 4 if c["src"] == "f32" else 2
    row = K * (D + 1 if c["cache"] == "e4m3" else 2 * D)  # bytes of one position's keys (or values)
    index = 4 * (2 * B + 1) + 4 * sum(-(-(a + n) // c["page"]) for a, n in zip(cached, new))
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(cached, new))
    if c["op"] == "rope":
        return {"bytes": 2 * T * H * D * src + 4 * T, "flops": 3 * T * H * c["rot"]}
    if c["op"] == "append":
        return {"bytes": T * (H + 2 * K) * D * src + 2 * T * H * D + 2 * T * row + index,
                "flops": 3 * T * (H + K) * c["rot"]}
    if c["op"] == "read":
        return {"bytes": 2 * T * (row + 2 * K * D) + index, "flops": 2 * T * K * D if c["cache"] == "e4m3" else 0}
    if c["op"] == "paged":
        return {"bytes": 4 * T * H * D + 2 * sum(a + n for a, n in zip(cached, new)) * row + index,
                "flops": 4 * D * H * pairs}
    return {"bytes": 2 * T * (2 * H + 2 * K) * D + 4 * (B + 1), "flops": 4 * D * H * pairs}


# ---- the same in 64 bits -------------------------------------------------------------------


def _turn64(x, positions, case):
    """Rows rotated as complex numbers."""
    inv, m = _inv_freq(case)
    turn = torch.polar(torch.full((), m, dtype=torch.float64, device=DEV), positions.double()[:, None] * inv)[:, None]
    rot, x = case["rot"], x.double()
    r = x[..., :rot]
    r = r.unflatten(-1, (-1, 2)) if case["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(r.contiguous()) * turn)
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., rot:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    new, cached = _ints(c["new"]), _ints(c["cached"])
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(cached, new)]).to(DEV)
    if c["op"] == "rope":
        return _turn64(s["x"], pos, c)
    if c["op"] == "append":
        # what the written pages stand for before their rounding: bf16 rows, or codes under the
        # row's power of two (which has no 64-bit value of its own)
        k, v = _turn64(s["k"], pos, c), s["v"].double()
        seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
        page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
        got = {"q": _turn64(s["q"], pos, c)}
        for name, x, limit in (("k", k, _limit(c)), ("v", v, 448.0)):
            pool = s[name + "_pages"].double()
            if c["cache"] == "e4m3":
                x = x * torch.exp2(-_exponent(s[name].float().abs().amax(-1), limit).double())[..., None]
                got[name + "_exp"] = None
            pool[page, :, slot] = x
            got[name] = pool
        return got
    if c["op"] == "read":
        return [torch.cat([_values(s, name, torch.float64)[s["table"][b].long()].transpose(1, 2).flatten(0, 1)[a:a + n]
                           for b, (a, n) in enumerate(zip(cached, new))]) for name in ("k", "v")]
    out, at = [], 0
    H, K = c["heads"], c["kv_heads"]
    for b, (a, n) in enumerate(zip(cached, new)):
        if c["op"] == "paged":
            k, v = (_values(s, name, torch.float64)[s["table"][b].long()].transpose(1, 2).flatten(0, 1)[:a + n]
                    for name in ("k", "v"))
        else:
            k, v = s["k"][at:at + n].double(), s["v"][at:at + n].double()
        q = s["q"][at:at + n].double()
        later = torch.arange(a + n, device=DEV)[None] > torch.arange(a, a + n, device=DEV)[:, None]
        one = torch.empty((n, H, c["head_dim"]), dtype=torch.float64, device=DEV)
        for h in range(H):
            w = (q[:, h] @ k[:, h // (H // K)].T * s["scale"]).masked_fill_(later, float("-inf")).softmax(-1)
            one[:, h] = w @ v[:, h // (H // K)]
        out.append(one)
        at += n
    return torch.cat(out)
