"""The serving operators: what is measured of them.

Attention with a sliding window and first tokens that stay visible ("window"),
attention over a paged cache held in 4 bits ("attend"), the quantising write to
that cache ("append"), block tables and slots from request lengths ("plan"),
and the norm of queries and keys with the position rotation ("rotary").

``run`` computes an operator in its plain form while ``own`` is false, and
through the package's entry points where it is true.  ``exact`` computes the
same from the definitions in 64 bits.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the prompt of one long request, 32 query heads over 8 key heads
        dict(name="window prompt", op="window", form="dense", batch=1, heads=32, kv_heads=8, n=8192, m=8192, dim=128,
             value_dim=128, window=1024, sinks=4, dtype="bfloat16"),
        # this framework's own type and head width, every query head with its own keys
        dict(name="window float32", op="window", form="dense", batch=2, heads=8, kv_heads=8, n=4096, m=4096, dim=64,
             value_dim=64, window=512, sinks=16, dtype="float32"),
        # a ragged batch of prompts, some of them continued behind keys of an earlier part; a head width of no power of two
        dict(name="window ragged", op="window", form="packed", batch=13, heads=8, kv_heads=2, n=411, m=623, dim=80,
             value_dim=80, window=300, sinks=1, dtype="float16"),
        # one new token of each of 16 requests
        dict(name="window one token", op="window", form="dense", batch=16, heads=32, kv_heads=8, n=1, m=4096, dim=128,
             value_dim=128, window=4096, sinks=0, dtype="bfloat16"),
        # a full serving batch over long requests, nothing hidden
        dict(name="attend batch", op="attend", requests=64, heads=32, kv_heads=8, n=1, length=12000, dim=128, page=64,
             window=0, sinks=0, dtype="bfloat16"),
        # one request, three tokens at once, float32, window and first tokens: latency
        dict(name="attend one request", op="attend", requests=1, heads=8, kv_heads=4, n=3, length=5000, dim=64, page=16,
             window=2048, sinks=4, dtype="float32"),
        # a decode step's new tokens
        dict(name="append step", op="append", tokens=48, kv_heads=8, dim=128, page=64, pages=128, padding=16,
             dtype="bfloat16"),
        # a prompt's tokens
        dict(name="append prompt", op="append", tokens=20011, kv_heads=8, dim=128, page=64, pages=512, padding=0,
             dtype="bfloat16"),
        # a decode step of a small batch: one token each
        dict(name="plan step", op="plan", requests=24, length=3000, new=1, page=16, width=512),
        # the prompts of a large batch
        dict(name="plan prompts", op="plan", requests=1000, length=900, new=400, page=64, width=64),
        # queries and keys of a decode step
        dict(name="rotary step", op="rotary", tokens=24, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             dtype="bfloat16"),
        # queries and keys of a prompt
        dict(name="rotary prompt", op="rotary", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["window", "window", "attend", "attend", "append", "plan", "rotary"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    group = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, rng.randint(17, 128)])
    if op == "window":
        form = rng.choice(["dense", "dense", "packed"])
        kv_heads = rng.choice([1, 2, 4, 8])
        batch = rng.randint(1, 4) if form == "dense" else rng.randint(1, 24)
        n = rng.choice([1, _spread(rng, 1, 4096), _spread(rng, 64, 4096)])
        m = n + rng.choice([0, 0, _spread(rng, 1, 4096)])
        # the plain form keeps every score of every head: at most as many as the largest listed case has
        room = (32 * 8192 * 8192) / (batch * kv_heads * group * (1 if form == "dense" else batch))
        n = max(1, min(n, int(math.sqrt(room))))
        m = max(n, min(m, int(room / n)))
        return dict(op=op, form=form, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, n=n, m=m, dim=dim,
                    value_dim=rng.choice([dim, dim, dim, 64]), window=_spread(rng, 1, 4096),
                    sinks=rng.choice([0, 1, 4, rng.randint(0, 200)]), dtype=dtype)
    if op == "attend":
        requests = _spread(rng, 1, 64)
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([dim, dim, 256])
        length = min(_spread(rng, 16, 40000), 64 * 12000 * 8 * 128 // (requests * kv_heads * max(dim, 32) * 2))
        return dict(op=op, requests=requests, heads=kv_heads * group, kv_heads=kv_heads, n=rng.choice([1, 1, 1, 2, 5]),
                    length=max(16, length), dim=dim, page=rng.choice([16, 32, 64, 128]),
                    window=rng.choice([0, _spread(rng, 16, 8192)]), sinks=rng.choice([0, 4, rng.randint(0, 100)]),
                    dtype=dtype)
    if op == "append":
        tokens = _spread(rng, 1, 20000)
        page = rng.choice([16, 32, 64, 128])
        return dict(op=op, tokens=tokens, kv_heads=rng.choice([1, 2, 4, 8]), dim=dim, page=page,
                    pages=tokens // page + rng.randint(1, 200), padding=rng.choice([0, rng.randint(1, 64)]), dtype=dtype)
    if op == "plan":
        return dict(op=op, requests=_spread(rng, 1, 1000), length=_spread(rng, 1, 2000),
                    new=rng.choice([1, _spread(rng, 1, 400)]), page=rng.choice([16, 32, 64, 128]),
                    width=rng.choice([160, 256, 333]))
    half = max(1, dim // 2)
    return dict(op=op, tokens=_spread(rng, 1, 16384), heads=rng.choice([4, 8, 16, 32]), kv_heads=rng.choice([1, 2, 4, 8]),
                dim=dim, rotary=2 * rng.choice([half, half, max(1, half // 2)]), interleaved=rng.random() < 0.3,
                dtype=dtype)


def _lengths(case):
    """Of a packed case, each request's new tokens and keys (a request keeps at least one of each); from the case alone."""
    r = np.random.RandomState(case["batch"] * 7919 + case["n"] * 31 + case["m"])
    n = np.maximum(1, np.ceil(r.random_sample(case["batch"]) * case["n"])).astype(np.int64)
    m = n + np.ceil(r.random_sample(case["batch"]) * (case["m"] - case["n"])).astype(np.int64)
    return n, m


def _held(case):
    """Of an attend case, each request's tokens, the new ones among them; from the case alone."""
    r = np.random.RandomState(case["requests"] * 7919 + case["length"])
    return np.maximum(case["n"], np.ceil((0.5 + 0.5 * r.random_sample(case["requests"])) * case["length"])).astype(np.int64)


def _padded_dim(dim):
    """Width of a row of codes: the head width filled up to 32, 64, 128 or 256."""
    return max(32, 1 << (dim - 1).bit_length())


def _visible(last, window, sinks):
    """How many keys the query at position `last` sees (0: a window without end)."""
    if window <= 0 or last + 1 <= window:
        return last + 1
    return window + min(sinks, last + 1 - window)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return dict(case=case, **_INPUTS[case["op"]](case, g))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _window_inputs(case, g):
    dt, d, dv = _TYPES[case["dtype"]], case["dim"], case["value_dim"]
    if case["form"] == "dense":
        q = _normal(g, (case["batch"], case["heads"], case["n"], d), dt, 1.5)
        k = _normal(g, (case["batch"], case["kv_heads"], case["m"], d), dt)
        v = _normal(g, (case["batch"], case["kv_heads"], case["m"], dv), dt)
        return dict(q=q, k=k, v=v)
    n, m = _lengths(case)
    cu_q = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device="cuda")
    cu_k = torch.tensor([0] + list(np.cumsum(m)), dtype=torch.int32, device="cuda")
    q = _normal(g, (int(n.sum()), case["heads"], d), dt, 1.5)
    k = _normal(g, (int(m.sum()), case["kv_heads"], d), dt)
    v = _normal(g, (int(m.sum()), case["kv_heads"], dv), dt)
    return dict(q=q, k=k, v=v, cu_q=cu_q, cu_k=cu_k)


def _attend_inputs(case, g):
    r, h, page, dp = case["requests"], case["kv_heads"], case["page"], _padded_dim(case["dim"])
    held = _held(case)
    need = -(-held // page)
    width, pages = int(need.max()), int(need.sum())
    # pages are handed out in any order; the entries behind a request's last page say nothing
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    row = torch.arange(width, device="cuda")[None, :]
    count = torch.tensor(need, device="cuda")[:, None]
    start = (torch.cumsum(count, 0) - count)
    tables = torch.where(row < count, order[(start + row).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))

    def codes(shape):
        return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)

    def params():
        # the scale and the least value of each row, as rows of roughly normal values have them
        scale = 0.25 + 0.15 * torch.rand((pages, h, page, 1), generator=g, device="cuda")
        least = -7.5 * scale + 0.3 * torch.randn((pages, h, page, 1), generator=g, device="cuda")
        return torch.cat([scale, least], -1).to(torch.bfloat16)

    q = _normal(g, (r, case["n"], case["heads"], case["dim"]), _TYPES[case["dtype"]], 1.5)
    return dict(q=q, k_codes=codes((pages, h, page, dp // 2)), k_params=params(),
                v_codes=codes((pages, h, page // 4, dp // 2, 4)), v_params=params(), tables=tables.contiguous(),
                lengths=torch.tensor(held, dtype=torch.int32, device="cuda"))


def _append_inputs(case, g):
    t, h, page, pages, dp = case["tokens"], case["kv_heads"], case["page"], case["pages"], _padded_dim(case["dim"])
    total = t + case["padding"]
    dt = _TYPES[case["dtype"]]
    # values as keys have them: some channels much larger than the others, each row with a level of its own
    channel = torch.exp(0.7 * torch.randn(case["dim"], generator=g, device="cuda"))
    k = (torch.randn((total, h, case["dim"]), generator=g, device="cuda") * channel).to(dt)
    v = (torch.randn((total, h, case["dim"]), generator=g, device="cuda")
         + 0.5 * torch.randn((total, h, 1), generator=g, device="cuda")).to(dt)
    # tokens fill whole pages one after another, the pages in any order; the padded tokens have no slot
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(t, device="cuda") % (pages * page)
    slots = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    slots[:t] = (order[at // page] * page + at % page).to(torch.int32)
    return dict(k=k, v=v, slots=slots, k_codes=torch.zeros((pages, h, page, dp // 2), dtype=torch.uint8, device="cuda"),
                k_params=torch.zeros((pages, h, page, 2), dtype=torch.bfloat16, device="cuda"),
                v_codes=torch.zeros((pages, h, page // 4, dp // 2, 4), dtype=torch.uint8, device="cuda"),
                v_params=torch.zeros((pages, h, page, 2), dtype=torch.bfloat16, device="cuda"))


def _plan_inputs(case, g):
    r, page, width = case["requests"], case["page"], case["width"]
    lengths = torch.randint(0, min(case["length"], width * page - case["new"]) + 1, (r,), generator=g, device="cuda", dtype=torch.int32)
    if case["new"] == 1:
        new = (torch.rand(r, generator=g, device="cuda") < 0.9).to(torch.int32)
    else:
        new = torch.randint(0, case["new"] + 1, (r,), generator=g, device="cuda", dtype=torch.int32)
    held = (lengths.long() + page - 1) // page
    start = torch.cumsum(held, 0) - held
    pages = r * width
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    row = torch.arange(width, device="cuda")[None, :]
    tables = torch.where(row < held[:, None], order[(start[:, None] + row).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    used = held.sum()
    # the free pages stand at the front of their list
    free = order[(torch.arange(pages, device="cuda") + used) % pages].contiguous()
    count = (pages - used).to(torch.int32).reshape(1)
    return dict(lengths=lengths, new=new, tables=tables.contiguous(), free=free, count=count, max_tokens=r * case["new"] + 5)


def _rotary_inputs(case, g):
    dt, t, d = _TYPES[case["dtype"]], case["tokens"], case["dim"]
    # queries and keys are slices of the one projection of a layer
    qkv = _normal(g, (t, case["heads"] + 2 * case["kv_heads"], d), dt, 2.0)
    q, k = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + case["kv_heads"]]
    positions = torch.randint(0, 200000, (t,), generator=g, device="cuda", dtype=torch.int32)
    q_weight = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
    k_weight = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
    half = case["rotary"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return dict(q=q, k=k, positions=positions, q_weight=q_weight, k_weight=k_weight, frequencies=freq)


_INPUTS = {"window": _window_inputs, "attend": _attend_inputs, "append": _append_inputs, "plan": _plan_inputs,
           "rotary": _rotary_inputs}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state["case"], state)


# ---- the package's entry points

def _window_own(case, s):
    import streaming_attention_b200 as sa
    if case["form"] == "dense":
        return sa.sliding_window_attention(s["q"], s["k"], s["v"], window=case["window"], sinks=case["sinks"])
    return sa.sliding_window_attention_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], window=case["window"],
                                              sinks=case["sinks"])


def _cache_of(case, s):
    import streaming_attention_b200 as sa
    return sa.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], case["dim"])


def _attend_own(case, s):
    return _cache_of(case, s).attend(s["q"], s["tables"], s["lengths"], window=case["window"] or None, sinks=case["sinks"])


def _append_own(case, s):
    cache = _cache_of(case, s)
    cache.append(s["k"], s["v"], s["slots"])
    return cache.read(s["slots"])


def _plan_own(case, s):
    import streaming_attention_b200 as sa
    p = sa.plan_kv_pages(s["lengths"], s["new"], s["tables"], s["free"], s["count"], page_size=case["page"],
                         max_tokens=s["max_tokens"])
    return p.lengths, p.offsets, p.positions, p.slots, p.tables, p.free_count


def _rotary_own(case, s):
    import streaming_attention_b200 as sa
    return sa.qk_norm_rotary(s["q"], s["k"], s["positions"], s["q_weight"], s["k_weight"], s["frequencies"], eps=1e-6,
                             interleaved=case["interleaved"])


_OWN = {"window": _window_own, "attend": _attend_own, "append": _append_own, "plan": _plan_own, "rotary": _rotary_own}


# ---- the plain forms

def _softmax_product(scores, mask, v):
    """softmax over the visible scores times v; a row that sees nothing is zero."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.clamp(min=1e-30)


def _window_plain(case, s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    group, window, sinks = case["heads"] // case["kv_heads"], case["window"], case["sinks"]
    if case["form"] == "dense":
        b, n, m = case["batch"], case["n"], case["m"]
        at = (m - n + torch.arange(n, device="cuda"))[:, None]
        j = torch.arange(m, device="cuda")[None, :]
        mask = (j <= at) & ((j > at - window) | (j < sinks))
        q = q.reshape(b, case["kv_heads"], group, n, -1)
        scores = torch.matmul(q, k[:, :, None].transpose(-1, -2)) / math.sqrt(case["dim"])
        out = _softmax_product(scores, mask, v[:, :, None]).reshape(b, case["heads"], n, -1)
        return out.to(s["q"].dtype)
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    t = torch.arange(q.shape[0], device="cuda")
    u = torch.arange(k.shape[0], device="cuda")
    rq = torch.searchsorted(cu_q, t, right=True) - 1
    rk = torch.searchsorted(cu_k, u, right=True) - 1
    n, m = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    at = (t - cu_q[rq] + (m - n)[rq])[:, None]
    j = (u - cu_k[rk])[None, :]
    mask = (rq[:, None] == rk[None, :]) & (j <= at) & ((j > at - window) | (j < sinks))
    q = q.reshape(q.shape[0], case["kv_heads"], group, -1).permute(1, 2, 0, 3)
    scores = torch.matmul(q, k.permute(1, 2, 0)[:, None]) / math.sqrt(case["dim"])
    out = _softmax_product(scores, mask, v.permute(1, 0, 2)[:, None])
    return out.permute(2, 0, 1, 3).reshape(t.shape[0], case["heads"], -1).to(s["q"].dtype)


def _nibbles(codes):
    """The two codes of each byte, the low one first, along the last axis."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, params, dim):
    """What rows of codes [..., padded width] stand for."""
    p = params.float()
    return codes[..., :dim].float() * p[..., 0:1] + p[..., 1:2]


def _attend_plain(case, s):
    r, n, group, page, dim = case["requests"], case["n"], case["heads"] // case["kv_heads"], case["page"], case["dim"]
    at = s["tables"].long().clamp(min=0)
    h, width = case["kv_heads"], at.shape[1]
    kc = _nibbles(s["k_codes"][at].permute(0, 2, 1, 3, 4).reshape(r, h, width * page, -1))
    vc = s["v_codes"][at].permute(0, 2, 1, 3, 5, 4).reshape(r, h, width * page, -1)
    k = _values(kc, s["k_params"][at].permute(0, 2, 1, 3, 4).reshape(r, h, width * page, 2), dim)
    v = _values(_nibbles(vc), s["v_params"][at].permute(0, 2, 1, 3, 4).reshape(r, h, width * page, 2), dim)
    length = s["lengths"].long()[:, None, None]
    i = length - n + torch.arange(n, device="cuda")[None, :, None]
    j = torch.arange(width * page, device="cuda")[None, None, :]
    mask = (j <= i) & (j < length)
    if case["window"]:
        mask = mask & ((j > i - case["window"]) | (j < case["sinks"]))
    q = s["q"].float().reshape(r, n, h, group, dim).permute(0, 2, 3, 1, 4).reshape(r, h, group * n, dim)
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim)
    mask = mask[:, None, None].expand(r, 1, group, n, width * page).reshape(r, 1, group * n, width * page)
    out = _softmax_product(scores, mask, v)
    return out.reshape(r, h, group, n, dim).permute(0, 3, 1, 2, 4).reshape(r, n, case["heads"], dim).to(s["q"].dtype)


def _quantise(x, dp):
    """Rows of x as codes, scales and least values, the codes' borders decided in 64 bits."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    least = low.float().to(torch.bfloat16)
    scale = ((high - low) / 15.0).float().to(torch.bfloat16)
    s = scale.double()
    codes = torch.where(s > 0, torch.round((x - least.double()) / s.clamp(min=1e-300)), torch.zeros((), dtype=torch.float64, device=x.device))
    codes = codes.clamp(0, 15).to(torch.uint8)
    codes = torch.nn.functional.pad(codes, (0, dp - codes.shape[-1]))
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat([scale, least], -1)


def _append_plain(case, s):
    page, dim, dp = case["page"], case["dim"], _padded_dim(case["dim"])
    slots = s["slots"].long()
    held = slots >= 0
    at, off = slots[held] // page, slots[held] % page
    kc, kp = _quantise(s["k"], dp)
    vc, vp = _quantise(s["v"], dp)
    s["k_codes"].permute(0, 2, 1, 3)[at, off] = kc[held]
    s["k_params"].permute(0, 2, 1, 3)[at, off] = kp[held]
    s["v_codes"].permute(0, 2, 4, 1, 3)[at, off // 4, off % 4] = vc[held]
    s["v_params"].permute(0, 2, 1, 3)[at, off] = vp[held]
    # and read back what is held
    where, off = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    k = _values(_nibbles(s["k_codes"].permute(0, 2, 1, 3)[where, off]), s["k_params"].permute(0, 2, 1, 3)[where, off], dim)
    v = _values(_nibbles(s["v_codes"].permute(0, 2, 4, 1, 3)[where, off // 4, off % 4]), s["v_params"].permute(0, 2, 1, 3)[where, off], dim)
    none = ~held[:, None, None]
    return k.masked_fill(none, 0.0), v.masked_fill(none, 0.0)


def _plan_plain(case, s):
    page, width, cap = case["page"], s["tables"].shape[1], s["max_tokens"]
    lengths, new = s["lengths"].long(), s["new"].long()
    after = lengths + new
    offsets = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    had, has = (lengths + page - 1) // page, (after + page - 1) // page
    taken = torch.cumsum(has - had, 0)
    row = torch.arange(width, device="cuda")[None, :]
    place = s["count"].long() - 1 - (taken - (has - had))[:, None] - (row - had[:, None])
    fresh = (row >= had[:, None]) & (row < has[:, None])
    tables = torch.where(fresh, s["free"][place.clamp(0, s["free"].shape[0] - 1)], s["tables"])
    t = torch.arange(cap, device="cuda")
    request = (torch.searchsorted(offsets, t, right=True) - 1).clamp(max=lengths.shape[0] - 1)
    position = lengths[request] + t - offsets[request]
    held = t < offsets[-1]
    slot = tables[request, (position // page).clamp(max=width - 1)].long() * page + position % page
    minus = torch.full((), -1, device="cuda")
    i32 = torch.int32
    return (after.to(i32), offsets.to(i32), torch.where(held, position, minus).to(i32),
            torch.where(held, slot, minus).to(i32), tables, (s["count"].long() - taken[-1]).to(i32))


def _rotary_plain(case, s):
    half, d = case["rotary"] // 2, case["dim"]
    # angles of far positions need more than 32 bits
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))

    def one(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        out = y.clone()
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
        return out.to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


_PLAIN = {"window": _window_plain, "attend": _attend_plain, "append": _append_plain, "plan": _plan_plain,
          "rotary": _rotary_plain}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    size = {"float32": 4}.get(case.get("dtype"), 2)
    if op == "window":
        n, m = _lengths(case) if case["form"] == "packed" else (np.full(case["batch"], case["n"]), np.full(case["batch"], case["m"]))
        pairs = keys = 0
        for a, b in zip(n.tolist(), m.tolist()):
            pairs += sum(_visible(p, case["window"], case["sinks"]) for p in range(b - a, b))
            first = max(0, b - a - case["window"] + 1)
            keys += b - first + min(case["sinks"], first)
        d, dv = case["dim"], case["value_dim"]
        return {"bytes": size * (int(n.sum()) * case["heads"] * (d + dv) + keys * case["kv_heads"] * (d + dv)),
                "flops": 2 * pairs * case["heads"] * (d + dv)}
    if op == "attend":
        d, w, keys, pairs = case["dim"], case["window"], 0, 0
        for length in _held(case).tolist():
            pairs += sum(_visible(p, w, case["sinks"]) for p in range(length - case["n"], length))
            first = max(0, length - case["n"] - w + 1) if w else 0
            keys += length - first + min(case["sinks"], first)
        return {"bytes": keys * case["kv_heads"] * 2 * (d / 2 + 4) + 2 * size * case["requests"] * case["n"] * case["heads"] * d,
                "flops": 4 * pairs * case["heads"] * d}
    if op == "append":
        rows = case["tokens"] * case["kv_heads"] * 2
        # the values are read, the codes written and read, the values they stand for written
        return {"bytes": rows * (case["dim"] * size + 2 * (case["dim"] / 2 + 4) + 4 * case["dim"]), "flops": 8 * rows * case["dim"]}
    if op == "plan":
        tokens = case["requests"] * case["new"]
        return {"bytes": 16 * case["requests"] + 8 * tokens + 8 * (tokens // case["page"]), "flops": 0}
    rows = case["tokens"] * (case["heads"] + case["kv_heads"])
    return {"bytes": 2 * rows * case["dim"] * size, "flops": 8 * rows * case["dim"]}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _attention64(q, k, v, sees):
    """One request: q [h, n, d], k [h, m, d], v [h, m, dv], sees [n, m]."""
    x = torch.einsum("hnd,hmd->hnm", q, k) / math.sqrt(q.shape[-1])
    x = torch.where(sees, x, torch.full((), -math.inf, dtype=torch.float64, device=x.device))
    w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    return torch.einsum("hnm,hmd->hnd", w, v)


def _sees(n, m, window, sinks):
    at = torch.arange(m - n, m, device="cuda").unsqueeze(1)
    j = torch.arange(m, device="cuda").unsqueeze(0)
    near = torch.ones_like(j <= at) if not window else (at - j) < window
    return (at >= j) & (near | (j < sinks))


def _exact_window(case, s):
    heads, per = case["heads"], case["heads"] // case["kv_heads"]
    if case["form"] == "dense":
        out = torch.empty(case["batch"], heads, case["n"], case["value_dim"], dtype=torch.float64, device="cuda")
        sees = _sees(case["n"], case["m"], case["window"], case["sinks"])
        for b in range(case["batch"]):
            for h in range(heads):
                out[b, h] = _attention64(*(x.double() for x in (s["q"][b, h:h + 1], s["k"][b, h // per:h // per + 1], s["v"][b, h // per:h // per + 1])), sees)[0]
        return out
    n, m = _lengths(case)
    out, a, c = [], 0, 0
    for x, y in zip(n.tolist(), m.tolist()):
        k = s["k"][c:c + y].double().repeat_interleave(per, 1).transpose(0, 1)
        v = s["v"][c:c + y].double().repeat_interleave(per, 1).transpose(0, 1)
        out.append(_attention64(s["q"][a:a + x].double().transpose(0, 1), k, v, _sees(x, y, case["window"], case["sinks"])).transpose(0, 1))
        a, c = a + x, c + y
    return torch.cat(out)


def _row64(codes, params, dim):
    digit = torch.arange(codes.shape[-1] * 2, device="cuda")
    byte = codes.long()[..., digit // 2]
    return (((byte >> (4 * (digit % 2))) & 15).double() * params[..., :1].double() + params[..., 1:].double())[..., :dim]


def _exact_attend(case, s):
    per, page, n = case["heads"] // case["kv_heads"], case["page"], case["n"]
    out = []
    for r, length in enumerate(_held(case).tolist()):
        token = torch.arange(length, device="cuda")
        at, off = s["tables"][r].long()[token // page], token % page
        k = _row64(s["k_codes"][at, :, off], s["k_params"][at, :, off], case["dim"])
        v = _row64(s["v_codes"][at, :, off // 4, :, off % 4], s["v_params"][at, :, off], case["dim"])
        k, v = (x.repeat_interleave(per, 1).transpose(0, 1) for x in (k, v))
        out.append(_attention64(s["q"][r].double().transpose(0, 1), k, v, _sees(n, length, case["window"], case["sinks"])).transpose(0, 1))
    return torch.stack(out)


def _exact_append(case, s):
    def one(x):
        x = x.double()
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        m = low.to(torch.float32).to(torch.bfloat16).double()
        w = ((high - low) / 15).to(torch.float32).to(torch.bfloat16).double()
        code = torch.nan_to_num((x - m) / w, nan=0.0, posinf=15.0, neginf=0.0).round().clamp(0, 15)
        return torch.where((s["slots"] >= 0)[:, None, None], code * w + m, torch.zeros_like(x))

    return one(s["k"]), one(s["v"])


def _exact_rotary(case, s):
    half, d = case["rotary"] // 2, case["dim"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["frequencies"][None])[:, None]

    def one(x, w):
        y = x.double()
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / d + 1e-6) * w.double()
        head, rest = y[..., :2 * half], y[..., 2 * half:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, rest], -1)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def exact(case, seed):
    if case["op"] == "plan":
        return None     # whole numbers only
    one = {"window": _exact_window, "attend": _exact_attend, "append": _exact_append, "rotary": _exact_rotary}
    return one[case["op"]](case, prepare(case, seed))
