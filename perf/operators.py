"""What is measured of the serving-step operators: page allocation and release, per-head norms with rotation and cache
append, attention over a 4-bit paged cache.

``own`` false: the operators in elementary torch operations, in 32 bits (64 for keys that become codes, where a value next
to a rounding border must not depend on the order of a sum).  ``own`` true: the framework's operators.

The 4-bit cache holds blocks of 32 consecutive head elements as e2m1 codes (two to a byte, the lower nibble first) with one
power-of-two scale byte (exponent + 127) each: codes ``[pages, heads_kv, page_size, dim / 2]``, scales
``[pages, heads_kv, page_size, dim / 32]``.
"""

import functools
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's bookkeeping: 64 sequences of up to 8 K tokens, one new token each
        {"name": "alloc decode 64", "op": "alloc", "batch": 64, "page_size": 64, "max_len": 8192, "max_new": 1, "share": 1.0},
        # a prefill step: 33 ragged prompts of up to 8 K tokens on 16-token pages, the pool too small for the last of them
        {"name": "alloc prefill 33 ragged", "op": "alloc", "batch": 33, "page_size": 16, "max_len": 16384, "max_new": 8192, "share": 0.9},
        # finished requests of one step give their pages back
        {"name": "release 64", "op": "release", "batch": 64, "page_size": 64, "max_len": 8192, "finished": 0.2},
        # the end of a large batch of long requests on small pages
        {"name": "release 515 long", "op": "release", "batch": 515, "page_size": 16, "max_len": 16384, "finished": 0.7},
        # decode step of 64 sequences, Llama-3-8B heads, 4-bit cache, q/k/v as slices of one projection
        {"name": "append decode fp4", "op": "append", "tokens": 64, "pad": 3, "heads": 32, "heads_kv": 8, "dim": 128, "page_size": 64,
         "cache": "fp4", "dtype": "bfloat16", "rotary_dim": 128, "interleaved": False, "norm": True, "fused": True},
        # prefill chunks of 8 x 1024 tokens into the 4-bit cache
        {"name": "append prefill fp4", "op": "append", "tokens": 8192, "pad": 0, "heads": 32, "heads_kv": 8, "dim": 128, "page_size": 64,
         "cache": "fp4", "dtype": "bfloat16", "rotary_dim": 128, "interleaved": False, "norm": True, "fused": True},
        # odd token count, partial rotation of neighbouring pairs, FP8 cache with a scale per token and head, half precision
        {"name": "append 4099 fp8 half", "op": "append", "tokens": 4099, "pad": 5, "heads": 16, "heads_kv": 4, "dim": 64, "page_size": 16,
         "cache": "fp8", "dtype": "float16", "rotary_dim": 32, "interleaved": True, "norm": True, "fused": False},
        # wide heads, 16-bit cache, keys and queries rotated without a norm
        {"name": "append 2050 wide 16-bit", "op": "append", "tokens": 2050, "pad": 0, "heads": 16, "heads_kv": 2, "dim": 256, "page_size": 32,
         "cache": "same", "dtype": "bfloat16", "rotary_dim": 256, "interleaved": False, "norm": False, "fused": True},
        # one short request: latency
        {"name": "attend 1 x 300", "op": "attend", "batch": 1, "q_len": 1, "heads": 32, "heads_kv": 8, "dim": 128, "page_size": 16,
         "lo": 300, "hi": 300, "dtype": "float16", "softcap": 0.0},
        # a decode step of 64 sequences of 512 to 8192 tokens, Llama-3-8B heads
        {"name": "attend 64 ragged", "op": "attend", "batch": 64, "q_len": 1, "heads": 32, "heads_kv": 8, "dim": 128, "page_size": 64,
         "lo": 512, "hi": 8192, "dtype": "bfloat16", "softcap": 0.0},
        # long contexts: 8 sequences of 131072 tokens
        {"name": "attend 8 x 128k", "op": "attend", "batch": 8, "q_len": 1, "heads": 64, "heads_kv": 8, "dim": 128, "page_size": 64,
         "lo": 131072, "hi": 131072, "dtype": "bfloat16", "softcap": 0.0},
        # eight query tokens a sequence (verification of a draft), causal within them, capped scores
        {"name": "attend 32 x 8 tokens", "op": "attend", "batch": 32, "q_len": 8, "heads": 64, "heads_kv": 8, "dim": 128, "page_size": 64,
         "lo": 1024, "hi": 16384, "dtype": "bfloat16", "softcap": 30.0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["alloc", "release", "append", "append", "attend", "attend"])
    dtype, page = rng.choice(["bfloat16", "float16"]), rng.choice([16, 32, 64, 128])
    if op == "alloc":
        max_len = page * _spread(rng, 4, 16384 // page)
        batch = _spread(rng, 1, 600)
        return {"op": op, "batch": batch, "page_size": page, "max_len": max_len, "share": rng.choice([0.5, 0.9, 1.0, 1.0]),
                "max_new": rng.choice([1, _spread(rng, 1, max(1, min(max_len, 270000 // batch)))])}
    if op == "release":
        return {"op": op, "batch": _spread(rng, 1, 515), "page_size": page, "max_len": page * _spread(rng, 1, 16384 // page),
                "finished": rng.choice([0.02, 0.3, 0.7, 1.0])}
    heads_kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([64, 128, 128, 256])
    if op == "append":
        most = 8192 * 48 * 128 // (heads_kv * (group + 2) * dim)
        tokens = _spread(rng, 1, min(8192, most))
        rot = rng.choice([dim, dim, dim // 2, 32, 24, 0])
        norm = rng.choice([True, True, False])
        return {"op": op, "tokens": tokens, "pad": rng.choice([0, 0, min(7, tokens - 1)]), "heads": heads_kv * group, "heads_kv": heads_kv,
                "dim": dim, "page_size": page, "cache": rng.choice(["fp4", "fp4", "fp8", "same"]), "dtype": dtype, "rotary_dim": rot,
                "interleaved": rng.choice([False, False, True]), "norm": norm, "fused": rng.choice([True, False])}
    q_len = rng.choice([1, 1, 1, 2, 3, 8, 17])
    most = min(2 ** 29 // (heads_kv * dim), 2 ** 34 // (q_len * heads_kv * group * dim))  # tokens of context in all
    hi = _spread(rng, 1, min(131072, most))
    lo = rng.choice([hi, max(1, hi // 16), 0])
    batch = _spread(rng, 1, max(1, min(256, most // hi)))
    return {"op": op, "batch": batch, "q_len": q_len, "heads": heads_kv * group, "heads_kv": heads_kv, "dim": dim, "page_size": page,
            "lo": lo, "hi": hi, "dtype": dtype, "softcap": rng.choice([0.0, 0.0, 30.0])}


# --------------------------------------------------------------------------------------------------------------- 4 bits
# (written in elementary operations; torch.round goes to even, which is the tie rule of e2m1)
def _fp4_quantize(x):
    """``x [..., dim]`` in 32 bits -> (codes ``[..., dim / 2]`` uint8, scale bytes ``[..., dim / 32]`` uint8, the values in 32 bits)."""
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    mant, expo = torch.frexp(blocks.abs().amax(-1))
    e = torch.where(mant <= 0.75, expo - 3, expo - 2).clamp(-126, 127)  # the smallest e with amax <= 6 * 2^e
    e = torch.where(mant == 0, torch.full_like(e, -126), e)
    a = torch.ldexp(blocks, -e[..., None]).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = torch.round(a / step) * step
    index = torch.where(r < 2, 2 * r, torch.where(r < 4, r + 2, r * 0.5 + 4)).to(torch.uint8)
    code = (index | (torch.signbit(blocks).to(torch.uint8) << 3)).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    value = torch.ldexp(torch.where(torch.signbit(blocks), -r, r), e[..., None]).reshape(x.shape)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8), value


@functools.lru_cache(maxsize=None)
def _fp4_pairs(device, dtype):
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=device)
    v = torch.cat([v, -v])
    byte = torch.arange(256, device=device)
    return torch.stack([v[byte & 15], v[byte >> 4]], -1)


def _fp4_values(codes, scales, dtype=torch.float32):
    x = _fp4_pairs(codes.device, dtype)[codes.int()].reshape(*codes.shape[:-1], scales.shape[-1], 32)
    return (x * torch.exp2(scales.to(dtype) - 127)[..., None]).reshape(*codes.shape[:-1], codes.shape[-1] * 2)


# -------------------------------------------------------------------------------------------------------------- prepare
def _pages(lens, page):
    return (lens + page - 1) // page


def _tables(g, lens, width, page, spare, device, pool=None):
    """Block tables of sequences of ``lens`` tokens over one permuted pool (of just their pages and the spare ones, if no size is given),
    ``spare`` pages that none of them holds, and the pool's size."""
    n = _pages(lens, page)
    used = int(n.sum())
    pool = used + spare if pool is None else pool
    perm = torch.randperm(pool, generator=g, device=device).to(torch.int32)
    first = torch.cumsum(n, 0) - n
    lp = torch.arange(width, device=device)
    table = torch.where(lp < n[:, None], perm[(first[:, None] + lp).clamp(max=pool - 1)], 0).to(torch.int32)
    return table, perm[used:used + spare], pool


def _lens(g, lo, hi, n, device):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    return {"alloc": _prepare_pool, "release": _prepare_pool, "append": _prepare_append, "attend": _prepare_attend}[case["op"]](case, g, device)


def _prepare_pool(case, g, device):
    batch, page, width = case["batch"], case["page_size"], _pages(case["max_len"], case["page_size"])
    pool = batch * (width + 1)
    free_pages = torch.zeros(pool, dtype=torch.int32, device=device)
    state = {"case": case, "pool": pool, "width": width, "free_pages": free_pages}
    if case["op"] == "release":
        lens = _lens(g, 0, case["max_len"], batch, device)
        state["finished"] = torch.rand(batch, generator=g, device=device) < case["finished"]
        spare = batch
    else:
        total = max(1, batch * case["max_new"] // 2) if case["max_new"] > 1 else batch  # the step's token buffer, padded behind the last chunk
        new = _lens(g, 0, case["max_new"], batch, device) if case["max_new"] > 1 else torch.ones(batch, dtype=torch.int64, device=device)
        new = torch.where(new.sum() > total, new * total // new.sum().clamp(min=1), new)
        lens = (torch.rand(batch, generator=g, device=device) * (case["max_len"] - new + 1)).long()
        spare = max(1, int(math.ceil(case["share"] * int((_pages(lens + new, page) - _pages(lens, page)).sum()))))
        state["cu"] = None if case["max_new"] == 1 else torch.cat([new.new_zeros(1), torch.cumsum(new, 0)]).int()
        state["total"] = total
    state["table"], free_pages[:spare], _ = _tables(g, lens, width, page, spare, device, pool)
    return {**state, "lens": lens.int(), "free_count": torch.tensor([spare], dtype=torch.int32, device=device)}


def _prepare_append(case, g, device):
    t, h, hk, d, page, dtype = case["tokens"], case["heads"], case["heads_kv"], case["dim"], case["page_size"], DTYPES[case["dtype"]]
    randn = functools.partial(torch.randn, generator=g, device=device)
    if case["fused"]:  # slices of one projection's output
        qkv = randn(t, (h + 2 * hk) * d).to(dtype)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, hk * d, hk * d], 1))
    else:
        q, k, v = (randn(t, n, d).to(dtype) for n in (h, hk, hk))
    pages = _pages(t, page) + 7
    order = torch.randperm(pages, generator=g, device=device)
    token = torch.arange(t, device=device)
    slots = order[token // page] * page + token % page
    valid = t - case["pad"]
    slots[valid:] = -1
    base = int(torch.randint(0, 65536 - t, (1,), generator=g, device=device))
    half = case["rotary_dim"] // 2
    state = {"case": case, "q": q, "k": k, "v": v, "slots": slots, "positions": (base + token).int(), "valid": valid,
             "q_weight": None, "k_weight": None, "cos": None, "sin": None, "k_scale": None, "v_scale": None}
    if case["norm"]:
        state["q_weight"], state["k_weight"] = ((1 + 0.2 * randn(d)).to(dtype) for _ in range(2))
    if half:
        angle = torch.arange(65536, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    for name in ("k", "v"):
        if case["cache"] == "fp4":
            state[name + "_cache"] = torch.zeros(pages, hk, page, d // 2, dtype=torch.uint8, device=device)
            state[name + "_scale"] = torch.ones(pages, hk, page, d // 32, dtype=torch.uint8, device=device)
        else:
            state[name + "_cache"] = torch.zeros(pages * page, hk, d, dtype=FP8 if case["cache"] == "fp8" else dtype, device=device)
            if case["cache"] == "fp8":
                state[name + "_scale"] = torch.ones(pages * page, hk, dtype=torch.float32, device=device)
    return state


def _prepare_attend(case, g, device):
    b, h, hk, d, page = case["batch"], case["heads"], case["heads_kv"], case["dim"], case["page_size"]
    hi = max(case["hi"], case["q_len"])
    lens = _lens(g, max(case["lo"], case["q_len"]) if case["lo"] else 0, hi, b, device)
    lens = torch.where(lens < case["q_len"], 0, lens)  # (a padded batch has sequences without tokens)
    table, _, pool = _tables(g, lens, _pages(hi, page), page, 3, device)
    shape = (b, h, d) if case["q_len"] == 1 else (b, case["q_len"], h, d)
    state = {"case": case, "q": torch.randn(shape, generator=g, device=device).to(DTYPES[case["dtype"]]), "lens": lens.int(), "table": table}
    step = max(1, (1 << 25) // (hk * page * d))  # the pool is drawn and rounded in portions
    for name in ("k", "v"):
        parts = [_fp4_quantize(torch.randn(min(step, pool - s), hk, page, d, generator=g, device=device))[:2] for s in range(0, pool, step)]
        state[name], state[name + "_scale"] = (torch.cat(x) for x in zip(*parts))
    return state


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    return {"alloc": _run_alloc, "release": _run_release, "append": _run_append, "attend": _run_attend}[state["case"]["op"]](state)


@functools.lru_cache(maxsize=None)
def _operator(name, *args, **kwargs):
    import tileops_amd

    return getattr(tileops_amd, name)(*args, **kwargs)


def _run_alloc(s):
    page, width, lens, table = s["case"]["page_size"], s["width"], s["lens"], s["table"]
    if own:
        op = _operator("PagedKVCacheAllocFwdOp", s["case"]["batch"], width, page, s["pool"])
        return (*op(lens, table, s["free_pages"], s["free_count"], s["cu"], s["total"]), table)
    cached, free_pages, free = lens.long(), s["free_pages"], s["free_count"].long()
    cu = torch.arange(len(lens) + 1, device=lens.device) if s["cu"] is None else s["cu"].long()
    new = cu[1:] - cu[:-1]
    before, after = _pages(cached, page), _pages(cached + new, page)
    fits = (cached + new <= width * page) & (new > 0)
    need = torch.where(fits, after - before, 0)
    last = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (last <= free))
    first = last - need
    lp = torch.arange(width, device=lens.device)
    fresh = free_pages[(free - 1 - (first[:, None] + lp - before[:, None])).clamp(0, s["pool"] - 1)]
    table.copy_(torch.where(served[:, None] & (lp >= before[:, None]) & (lp < after[:, None]), fresh, table))
    t = torch.arange(s["total"], device=lens.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=len(lens) - 1)
    pos = cached[b] + t - cu[b]
    good = (t < cu[-1]) & served[b]
    slots = table[b, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    taken = torch.where(served, need, 0).sum()
    return (torch.where(good, slots, -1), torch.where(good, pos, -1).int(), torch.where(served, cached + new, cached).int(),
            (new > 0) & ~served, (free - taken).int(), table)


def _run_release(s):
    page, lens, table, free_pages = s["case"]["page_size"], s["lens"], s["table"], s["free_pages"]
    if own:
        op = _operator("PagedKVCacheReleaseFwdOp", s["case"]["batch"], s["width"], page, s["pool"])
        return (*op(s["finished"], lens, table, free_pages, s["free_count"]), free_pages)
    n = torch.where(s["finished"], _pages(lens.long(), page), 0)
    first = torch.cumsum(n, 0) - n
    lp = torch.arange(s["width"], device=lens.device)
    to = torch.where(lp < n[:, None], s["free_count"].long() + first[:, None] + lp, s["pool"])
    grown = torch.cat([free_pages, free_pages[:1]])
    grown[to.reshape(-1)] = table.reshape(-1)
    free_pages.copy_(grown[:-1])
    return torch.where(s["finished"], 0, lens), (s["free_count"] + n.sum()).int(), free_pages


def _normed(x, weight, dtype):
    x = x.to(dtype)
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.to(dtype)


def _rotated(x, cos, sin, positions, interleaved):
    if cos is None:
        return x
    half = cos.shape[1]
    at = positions.long()
    c, s = cos[at].to(x.dtype)[:, None], sin[at].to(x.dtype)[:, None]
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    y = (a * c - b * s, b * c + a * s)
    return torch.cat([torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1), rest], -1)


def _run_append(s):
    c, n = s["case"], s["valid"]
    if own:
        kind = {"fp4": torch.float4_e2m1fn_x2, "fp8": FP8, "same": None}[c["cache"]]
        op = _operator("QKNormRopePagedKVAppendFwdOp", c["heads"], c["heads_kv"], c["dim"], c["page_size"], rotary_dim=c["rotary_dim"], eps=1e-6,
                       interleaved=c["interleaved"], cache_dtype=kind)
        q = op(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
               s["k_scale"], s["v_scale"])
        if c["cache"] == "fp4":  # the rows as the values that they stand for
            return (q, *_operator("PagedFP4KVCacheGatherFwdOp", c["heads_kv"], c["dim"], c["page_size"])(
                s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"][:n]))
        return q, s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]
    q = _rotated(_normed(s["q"], s["q_weight"], torch.float32), s["cos"], s["sin"], s["positions"], c["interleaved"]).to(s["q"].dtype)
    k = _rotated(_normed(s["k"], s["k_weight"], torch.float64), s["cos"], s["sin"], s["positions"], c["interleaved"]).float()[:n]
    store = _stored if c["cache"] == "fp4" else _pooled
    return (q, *store(s, "k", k), *store(s, "v", s["v"][:n].float()))


def _stored(s, name, x):
    codes, scales, values = _fp4_quantize(x)
    at, page = s["slots"][: s["valid"]], s["case"]["page_size"]
    s[name + "_cache"][at // page, :, at % page] = codes
    s[name + "_scale"][at // page, :, at % page] = scales
    return (values.bfloat16(),)


def _pooled(s, name, x):
    at = s["slots"][: s["valid"]]
    if s["case"]["cache"] == "fp8":
        scale = x.abs().amax(-1).clamp(min=1e-4) / 448.0
        s[name + "_scale"][at] = scale
        x = (x / scale[..., None]).clamp(-448.0, 448.0)
    s[name + "_cache"][at] = x.to(s[name + "_cache"].dtype)
    return s[name + "_cache"], s[name + "_scale"]


def _run_attend(s):
    c, q, lens, table = s["case"], s["q"], s["lens"], s["table"]
    b, hk, d, ql = c["batch"], c["heads_kv"], c["dim"], c["q_len"]
    if own:
        op = _operator("GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp", b, c["heads"], hk, s["k"].shape[0] * c["page_size"], d, c["page_size"],
                       q_len=ql, softcap=c["softcap"])
        return op(q, s["k"], s["v"], s["k_scale"], s["v_scale"], lens, table)
    group = c["heads"] // hk
    at = table.long()
    k, v = (_fp4_values(s[n][at], s[n + "_scale"][at]).transpose(1, 2).flatten(2, 3) for n in ("k", "v"))  # [b, hk, tokens, d]
    tokens = torch.arange(k.shape[2], device=q.device)
    there = tokens < lens[:, None]
    v = torch.where(there[:, None, :, None], v, 0)
    rows = q.float().reshape(b, ql, hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, ql * group, d)
    scores = torch.matmul(rows, k.transpose(2, 3)) * d ** -0.5
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    token_of = torch.arange(ql * group, device=q.device) // group
    seen = tokens[None, None, :] <= (lens[:, None] - ql + token_of)[:, :, None]  # bottom-right causal
    scores = torch.where(seen[:, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    return o.reshape(b, hk, ql, group, d).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "alloc":
        new = case["batch"] * (1 if case["max_new"] == 1 else case["max_new"] / 2)
        pages = new / case["page_size"]
        return {"bytes": new * 12 + pages * 8 + case["batch"] * 21, "flops": 0}
    if case["op"] == "release":
        return {"bytes": case["batch"] * (9 + case["finished"] * case["max_len"] / 2 / case["page_size"] * 8), "flops": 0}
    if case["op"] == "append":
        t, h, hk, d = (case[n] for n in ("tokens", "heads", "heads_kv", "dim"))
        row = {"fp4": d / 2 + d / 32, "fp8": d + 4, "same": 2 * d}[case["cache"]]
        angle = 4 * case["rotary_dim"]
        return {"bytes": t * ((2 * h + 2 * hk) * d * 2 + 2 * hk * row + angle + 12), "flops": t * (h + hk) * d * 8}
    lo = max(case["lo"], case["q_len"]) if case["lo"] else 0
    total = case["batch"] * (lo + max(case["hi"], case["q_len"])) / 2
    d, rows = case["dim"], case["batch"] * case["q_len"] * case["heads"]
    return {"bytes": total * case["heads_kv"] * 2 * (d / 2 + d / 32) + rows * d * 4, "flops": 4 * total * case["q_len"] * case["heads"] * d}


# ---------------------------------------------------------------------------------------------------------------- exact
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest_e2m1(x):
    """The values of e2m1 blocks with power-of-two scales that stand for ``x [..., dim]``: the nearest code, ties to the even one."""
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, 127.0)
    for _ in range(254):  # the smallest exponent from -126 up whose six times the scale reaches the largest value
        lower = (e > -126) & (amax <= 6 * torch.exp2(e - 1))
        if not bool(lower.any()):
            break
        e = torch.where(lower, e - 1, e)
    scale = torch.exp2(e)
    grid = torch.tensor(_E2M1, dtype=x.dtype, device=x.device)
    size = blocks.abs() / scale
    best, far = torch.zeros_like(size), size
    for i in range(1, 8):
        d = (size - grid[i]).abs()
        take = (d < far) | ((d == far) & (i % 2 == 0))
        best, far = torch.where(take, grid[i], best), torch.where(take, d, far)
    return (torch.sign(blocks) * best * scale).flatten(-2)


def exact(case, seed):
    if case["op"] in ("alloc", "release"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attend(s)


def _exact_head(x, weight, cos, sin, positions, interleaved):
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * weight.double()
    out = y.clone()
    if cos is not None:
        half = cos.shape[1]
        turn = torch.complex(cos.double(), sin.double())[positions.long()][:, None]
        lower, upper = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., lower], y[..., upper]) * turn
        out[..., lower], out[..., upper] = z.real, z.imag
    return out


def _exact_append(s):
    c, n = s["case"], s["valid"]
    q, k = (_exact_head(s[x], s[x + "_weight"], s["cos"], s["sin"], s["positions"], c["interleaved"]) for x in ("q", "k"))
    k, v = k[:n], s["v"][:n].double()
    if c["cache"] == "fp4":
        return q, _nearest_e2m1(k.float().double()), _nearest_e2m1(v)  # (keys are rounded to 32 bits once before the codes)
    out = [q]
    for name, x in (("k", k), ("v", v)):
        pool, scale = s[name + "_cache"].double(), None
        if c["cache"] == "fp8":
            scale = s[name + "_scale"].double()
            scale[s["slots"][:n]] = x.abs().amax(-1).clamp(min=1e-4) / 448
            x = x / scale[s["slots"][:n]][..., None]
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # of e4m3: three bits behind the leading one
            x = (torch.round(x / step) * step).clamp(-448, 448)
        pool[s["slots"][:n]] = x
        out += [pool, scale]
    return tuple(out)


def _exact_attend(s):
    c = s["case"]
    d, hk, ql, page = c["dim"], c["heads_kv"], c["q_len"], c["page_size"]
    group = c["heads"] // hk
    grid = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=s["q"].device)
    q = s["q"].double().reshape(c["batch"], ql, hk, group, d)
    out = torch.zeros_like(q)
    if c["batch"] * hk > 512:
        return None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, : _pages(n, page)].long()
        for h in range(hk):
            kv = []
            for name in ("k", "v"):
                byte = s[name][pages, h].reshape(-1, d // 2)[:n].long()
                x = torch.stack([grid[byte % 16], grid[byte // 16]], -1).reshape(n, d // 32, 32)
                scale = 2.0 ** (s[name + "_scale"][pages, h].reshape(-1, d // 32)[:n].double() - 127)
                kv.append((x * scale[..., None]).reshape(n, d))
            z = q[b, :, h].reshape(-1, d) @ kv[0].T.contiguous() / math.sqrt(d)
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            hidden = torch.arange(n, device=z.device)[None] > (n - ql + torch.arange(ql, device=z.device).repeat_interleave(group))[:, None]
            out[b, :, h] = (torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ kv[1]).reshape(ql, group, d)
    return out.reshape(s["q"].shape)
