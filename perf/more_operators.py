"""Long caches: what is measured of the operators that read or thin out the 4-bit
cache of long requests.

Attention of a batch that shares a long prefix ("shared"), the bounds of a
page's keys with the pages they select for each query ("select"), attention over
selected pages ("pages"), attention that accumulates the weight of every token
("weigh"), and eviction of the tokens of little weight ("evict").

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
        # a full serving batch behind one long document: one new token of each request
        dict(name="shared batch", op="shared", requests=64, heads=32, kv_heads=8, n=1, prefix=32000, length=400, dim=128,
             page=64, window=0, sinks=0, dtype="bfloat16"),
        # several tokens at once (a proposal being verified) behind a system prompt, a head width of no power of two
        dict(name="shared proposal", op="shared", requests=24, heads=16, kv_heads=2, n=4, prefix=5003, length=700, dim=80,
             page=32, window=0, sinks=0, dtype="float16"),
        # this framework's own type, with a window that ends inside the prefix for some requests, and first tokens
        dict(name="shared float32", op="shared", requests=9, heads=8, kv_heads=4, n=1, prefix=9000, length=900, dim=64,
             page=64, window=4096, sinks=4, dtype="float32"),
        # two requests behind a short prompt: latency
        dict(name="shared two", op="shared", requests=2, heads=8, kv_heads=8, n=1, prefix=333, length=50, dim=64, page=16,
             window=0, sinks=0, dtype="bfloat16"),
        # a decode step of a batch of long requests: the newest page's bounds, then the pages of each query
        dict(name="select batch", op="select", requests=48, heads=32, kv_heads=8, n=1, length=24000, new=1, dim=128,
             page=64, count=32, dtype="bfloat16"),
        # one request of many short pages after a part of its prompt: bounds of 2000 tokens, pages for three queries
        dict(name="select one request", op="select", requests=1, heads=8, kv_heads=4, n=3, length=9000, new=2000, dim=64,
             page=16, count=50, dtype="float32"),
        # the attention of the first of these two steps
        dict(name="pages batch", op="pages", requests=48, heads=32, kv_heads=8, n=1, length=24000, dim=128, page=64,
             count=32, dtype="bfloat16"),
        # and of the second
        dict(name="pages one request", op="pages", requests=1, heads=8, kv_heads=4, n=3, length=9000, dim=64, page=16,
             count=50, dtype="float32"),
        # a decode step of a batch whose tokens' weights are kept
        dict(name="weigh batch", op="weigh", requests=32, heads=32, kv_heads=8, n=1, length=10000, dim=128, page=64,
             window=0, sinks=0, dtype="bfloat16"),
        # one request, two tokens at once, a window with first tokens: latency
        dict(name="weigh one request", op="weigh", requests=1, heads=8, kv_heads=4, n=2, length=3000, dim=64, page=32,
             window=1024, sinks=4, dtype="float16"),
        # a batch where most requests have outgrown their limit
        dict(name="evict batch", op="evict", requests=48, kv_heads=8, length=8000, keep=2048, limit=4096, first=4,
             last=512, dim=128, page=64),
        # one request, a few tokens over
        dict(name="evict one request", op="evict", requests=1, kv_heads=4, length=1100, keep=777, limit=777, first=1,
             last=33, dim=64, page=16),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "shared", "select", "pages", "weigh", "evict"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    group = rng.choice([1, 2, 3, 4, 8])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, 256, rng.randint(17, 128)])
    page = rng.choice([16, 32, 64, 64, 128])
    case = dict(op=op, kv_heads=kv_heads, dim=dim, page=page)
    if op == "evict":
        requests = _spread(rng, 1, 48)
        # the largest listed case's tokens at most
        length = min(_spread(rng, 64, 16000), 48 * 8000 * 8 * 128 // (requests * kv_heads * max(dim, 32)))
        keep = max(8, int(length * rng.uniform(0.1, 0.8)))
        first = rng.choice([0, 1, 4, keep // 8])
        return dict(case, requests=requests, length=length, keep=keep, limit=rng.choice([keep, (keep + length) // 2]),
                    first=first, last=rng.randint(0, keep - first) // rng.choice([1, 4]))
    case.update(heads=kv_heads * group, dtype=dtype, n=rng.choice([1, 1, 1, 2, 5]))
    if op == "shared":
        requests = _spread(rng, 1, 64)
        rows = requests * case["n"] * case["heads"]
        prefix = min(_spread(rng, 1, 32000), 64 * 32 * 32000 * 128 // (rows * max(dim, 32)))
        length = min(_spread(rng, 1, 2000), 64 * 8 * 400 * 128 // (requests * kv_heads * max(dim, 32)))
        return dict(case, requests=requests, prefix=max(1, prefix), length=max(1, length),
                    window=rng.choice([0, 0, _spread(rng, 16, 8192)]), sinks=rng.choice([0, 4, rng.randint(0, 100)]))
    requests = _spread(rng, 1, 48)
    if op == "weigh":
        length = min(_spread(rng, 16, 40000), 32 * 10000 * 8 * 128 // (requests * kv_heads * max(dim, 32) * 2))
        return dict(case, requests=requests, length=max(16, length), window=rng.choice([0, 0, _spread(rng, 16, 8192)]),
                    sinks=rng.choice([0, 4, rng.randint(0, 100)]))
    room = 48 * 24000 * 8 * 128 // (requests * case["n"] * kv_heads * max(dim, 32) * 2)
    length = max(16, min(_spread(rng, 16, 60000), room))
    case.update(requests=requests, length=length, count=rng.choice([4, _spread(rng, 2, max(2, 2048 // page))]))
    if op == "select":
        case.update(new=rng.choice([1, _spread(rng, 1, max(1, length // 4))]))
    return case


def _padded_dim(dim):
    """Width of a row of codes: the head width filled up to 32, 64, 128 or 256."""
    return max(32, 1 << (dim - 1).bit_length())


def _held(case):
    """Tokens of each request (of "shared": its own ones); from the case alone."""
    r = np.random.RandomState(case["requests"] * 7919 + case["length"])
    part = 0.5 + 0.5 * r.random_sample(case["requests"])
    held = np.ceil(part * case["length"]).astype(np.int64)
    if case["op"] == "shared" and case["requests"] > 3:
        held[1] = 0   # an idle request: its rows are zero
        return held
    return np.maximum(case.get("n", 1), held)


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


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(case, g, need, spare=0):
    """The cache's four tensors, and tables of need[r] pages of any order; the entries
    behind a request's last page say nothing."""
    h, page, dp = case["kv_heads"], case["page"], _padded_dim(case["dim"])
    width, pages = int(need.max()), int(need.sum()) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    row = torch.arange(width, device="cuda")[None, :]
    count = torch.tensor(need, device="cuda")[:, None]
    start = torch.cumsum(count, 0) - count
    tables = torch.where(row < count, order[(start + row).clamp(max=pages - 1)], _i32(-1))

    def codes(shape):
        return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)

    def params():
        # the scale and the least value of each row, as rows of roughly normal values have them
        scale = 0.25 + 0.15 * torch.rand((pages, h, page, 1), generator=g, device="cuda")
        least = -7.5 * scale + 0.3 * torch.randn((pages, h, page, 1), generator=g, device="cuda")
        return torch.cat([scale, least], -1).to(torch.bfloat16)

    return dict(k_codes=codes((pages, h, page, dp // 2)), k_params=params(),
                v_codes=codes((pages, h, page // 4, dp // 2, 4)), v_params=params(), tables=tables.contiguous(), order=order)


def _queries(case, g):
    shape = (case["requests"], case["n"], case["heads"], case["dim"])
    return (1.5 * torch.randn(shape, generator=g, device="cuda")).to(_TYPES[case["dtype"]])


def _shared_inputs(case, g):
    held = _held(case)
    prefix_pages = -(-case["prefix"] // case["page"])
    s = _cache(case, g, np.concatenate([[prefix_pages], -(-held // case["page"])]))
    tables = s.pop("tables")
    width = max(1, int((-(-held // case["page"])).max()))
    return dict(s, q=_queries(case, g), prefix_table=tables[0].clone(), prefix_length=_i32([case["prefix"]]),
                tables=tables[1:, :width].contiguous(), lengths=_i32(held))


def _select_inputs(case, g):
    held = _held(case)
    s = _cache(case, g, -(-held // case["page"]))
    # bounds of every page as earlier steps left them
    dim, dp, shape = case["dim"], _padded_dim(case["dim"]), s["k_codes"].shape
    bounds = torch.zeros((*shape[:2], 2, dp), dtype=torch.bfloat16, device="cuda")
    mid = 0.3 * torch.randn((*shape[:2], dim), generator=g, device="cuda")
    bounds[..., 0, :dim] = (mid - 2.0 - 0.5 * torch.rand(mid.shape, generator=g, device="cuda")).to(torch.bfloat16)
    bounds[..., 1, :dim] = (mid + 2.0 + 0.5 * torch.rand(mid.shape, generator=g, device="cuda")).to(torch.bfloat16)
    return dict(s, q=_queries(case, g), bounds=bounds, lengths=_i32(held), new=_i32(np.minimum(case["new"], held)))


def _pages_inputs(case, g):
    held = _held(case)
    s = _cache(case, g, -(-held // case["page"]))
    # as a selection leaves them: ascending, the first page and the query's own among them, -1 behind
    r, n, h, count, width = case["requests"], case["n"], case["kv_heads"], case["count"], s["tables"].shape[1]
    i = torch.arange(n, device="cuda")
    last = (torch.tensor(held, device="cuda")[:, None] - n + i) // case["page"]           # [r, n]: the query's own page
    row = torch.arange(width, device="cuda")
    key = torch.rand((r, n, h, width), generator=g, device="cuda")
    key = torch.where(row == last[..., None, None], 3.0, torch.where(row == 0, 2.0, key))
    key = torch.where(row > last[..., None, None], -1.0, key)
    best = key.argsort(-1, descending=True)[..., :count]
    chosen = torch.where(best <= last[..., None, None], best, width).sort(-1).values
    pages = torch.full((r, n, h, count), -1, dtype=torch.int32, device="cuda")
    pages[..., :chosen.shape[-1]] = torch.where(chosen < width, chosen, -1).to(torch.int32)
    return dict(s, q=_queries(case, g), pages=pages, lengths=_i32(held))


def _weigh_inputs(case, g):
    held = _held(case)
    s = _cache(case, g, -(-held // case["page"]))
    # what earlier steps gave each token
    weights = torch.exp(2.0 * torch.randn(s["k_params"].shape[:3], generator=g, device="cuda") - 3.0)
    return dict(s, q=_queries(case, g), weights=weights, lengths=_i32(held))


def _evict_inputs(case, g):
    held, page = _held(case), case["page"]
    need = -(-held // page)
    s = _cache(case, g, need, spare=7)
    weights = torch.exp(2.0 * torch.randn(s["k_params"].shape[:3], generator=g, device="cuda") - 3.0)
    # tokens that no query has seen: equal weights
    weights = torch.where(torch.rand(weights.shape, generator=g, device="cuda") < 0.05, 0.0, weights)
    used, pages = int(need.sum()), s["order"].shape[0]
    free = s["order"][(torch.arange(pages, device="cuda") + used) % pages].contiguous()
    # the pages that an eviction writes to, as they were, so that a pass can be repeated
    kept = -(-case["keep"] // page)
    written = s["tables"][torch.tensor(held > case["limit"], device="cuda")][:, :kept].flatten().long()
    before = [s[x][written] for x in ("k_codes", "k_params", "v_codes", "v_params")]
    # and, for the values afterwards, the slots of what is kept at most
    token = torch.arange(case["keep"], device="cuda")
    entry = s["tables"][:, (token // page).clamp(max=s["tables"].shape[1] - 1)]
    slots = torch.where(token < torch.tensor(held, device="cuda")[:, None], entry * page + token % page, -1)
    return dict(s, weights=weights, lengths=_i32(held), free=free, count=_i32([pages - used]), written=written,
                before=before, slots=slots.to(torch.int32).flatten().contiguous())


_INPUTS = {"shared": _shared_inputs, "select": _select_inputs, "pages": _pages_inputs, "weigh": _weigh_inputs,
           "evict": _evict_inputs}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state["case"], state)


# ---- the package's entry points

def _cache_of(case, s):
    import streaming_attention_b200 as sa
    return sa.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], case["dim"])


def _shared_own(case, s):
    return _cache_of(case, s).attend_shared(s["q"], s["prefix_table"], s["prefix_length"], s["tables"], s["lengths"],
                                            window=case["window"] or None, sinks=case["sinks"])


def _select_own(case, s):
    cache = _cache_of(case, s)
    cache.update_page_bounds(s["bounds"], s["tables"], s["lengths"], s["new"])
    pages = cache.select_pages(s["q"], s["bounds"], s["tables"], s["lengths"], count=case["count"], first=1, last=1)
    return pages, s["bounds"]


def _pages_own(case, s):
    return _cache_of(case, s).attend_pages(s["q"], s["tables"], s["lengths"], s["pages"])


def _weigh_own(case, s):
    weights = s["weights"].clone()
    out = _cache_of(case, s).attend(s["q"], s["tables"], s["lengths"], window=case["window"] or None,
                                    sinks=case["sinks"], weights=weights)
    return out, weights


def _restored(s):
    """The state of an eviction as it was before it."""
    for x, y in zip(("k_codes", "k_params", "v_codes", "v_params"), s["before"]):
        s[x].index_copy_(0, s["written"], y)
    return s["weights"].clone(), s["lengths"].clone(), s["tables"].clone(), s["free"].clone(), s["count"].clone()


def _evict_own(case, s):
    weights, lengths, tables, free, count = _restored(s)
    cache = _cache_of(case, s)
    kept, dropped = cache.evict(weights, lengths, tables, free, count, keep=case["keep"], limit=case["limit"],
                                first=case["first"], last=case["last"])
    k, v = cache.read(s["slots"])
    return kept, dropped, lengths, tables, free, count, weights, k, v


_OWN = {"shared": _shared_own, "select": _select_own, "pages": _pages_own, "weigh": _weigh_own, "evict": _evict_own}


# ---- the plain forms

def _softmax(scores, mask):
    """softmax over the visible scores; a row that sees nothing is zero."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _nibbles(codes):
    """The two codes of each byte, the low one first, along the last axis."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, params, dim):
    """What rows of codes [..., padded width] stand for."""
    p = params.float()
    return codes[..., :dim].float() * p[..., 0:1] + p[..., 1:2]


def _tokens(case, s, at):
    """Keys and values of the pages `at` [..., w]: [..., heads, w * page, dim]."""
    at = at.long().clamp(min=0)
    page, dim = case["page"], case["dim"]

    def rows(x):
        return x.movedim(-3, -4).flatten(-3, -2)   # [..., w, heads, page, c] -> [..., heads, w * page, c]

    k = _values(_nibbles(rows(s["k_codes"][at])), rows(s["k_params"][at]), dim)
    v = s["v_codes"][at].transpose(-1, -2).flatten(-3, -2)   # [..., w, heads, page, bytes]
    return k, _values(_nibbles(rows(v)), rows(s["v_params"][at]), dim)


def _sees(position, j, window, sinks):
    sees = j <= position
    if window:
        sees = sees & ((j > position - window) | (j < sinks))
    return sees


def _grouped(case, q):
    """Queries [r, n, heads, dim] as [r, key heads, n * group, dim]."""
    r, n, h = case["requests"], case["n"], case["kv_heads"]
    return q.float().reshape(r, n, h, -1, case["dim"]).transpose(1, 2).reshape(r, h, -1, case["dim"])


def _ungrouped(case, out):
    r, n, h = case["requests"], case["n"], case["kv_heads"]
    return out.reshape(r, h, n, -1, case["dim"]).transpose(1, 2).reshape(r, n, case["heads"], case["dim"])


def _rows_mask(case, mask):
    """[r, n, m] -> [r, 1, n * group, m]."""
    return mask[:, None].repeat_interleave(case["heads"] // case["kv_heads"], 2)


def _shared_plain(case, s):
    n, scale = case["n"], 1.0 / math.sqrt(case["dim"])
    q = _grouped(case, s["q"])
    pk, pv = _tokens(case, s, s["prefix_table"])
    ok, ov = _tokens(case, s, s["tables"])
    length = s["lengths"].long()[:, None, None]
    own_position = length - n + torch.arange(n, device="cuda")[None, :, None]
    j = torch.arange(pk.shape[-2], device="cuda")
    u = torch.arange(ok.shape[-2], device="cuda")
    prefix = s["prefix_length"].long()
    position = prefix + own_position
    mask = torch.cat([(j < prefix) & _sees(position, j, case["window"], case["sinks"]),
                      (u < length) & _sees(position, prefix + u, case["window"], case["sinks"])], -1)
    mask = _rows_mask(case, mask & (own_position >= 0))
    scores = torch.cat([torch.matmul(q, pk.transpose(-1, -2)), torch.matmul(q, ok.transpose(-1, -2))], -1) * scale
    p = _softmax(scores, mask)
    out = torch.matmul(p[..., :pk.shape[-2]], pv) + torch.matmul(p[..., pk.shape[-2]:], ov)
    return _ungrouped(case, out).to(s["q"].dtype)


def _select_plain(case, s):
    r, n, h, page, dim, count = (case[x] for x in ("requests", "n", "kv_heads", "page", "dim", "count"))
    lengths, new, width = s["lengths"].long(), s["new"].long(), s["tables"].shape[1]
    # the bounds of the pages that the newest tokens stand in
    span = (case["new"] + page - 2) // page + 1
    at = ((lengths - new) // page)[:, None] + torch.arange(span, device="cuda")
    touched = (at * page < lengths[:, None]) & (new[:, None] > 0)
    at = torch.minimum(at, (lengths[:, None] - 1) // page).clamp(min=0)   # once more the last one, in place of none
    ids = torch.gather(s["tables"].long(), 1, at)
    k = _values(_nibbles(s["k_codes"][ids]), s["k_params"][ids], dim)                    # [r, span, h, page, dim]
    held = ((at * page)[..., None] + torch.arange(page, device="cuda") < lengths[:, None, None])[:, :, None, :, None]
    both = torch.stack([k.masked_fill(~held, math.inf).amin(-2), k.masked_fill(~held, -math.inf).amax(-2)], -2)
    was = s["bounds"][ids][..., :dim]
    s["bounds"][ids.flatten(), :, :, :dim] = torch.where(
        (touched | (new[:, None] > 0))[:, :, None, None, None], both.to(torch.bfloat16), was).flatten(0, 1)
    # scores in 64 bits: the pages must not depend on the order of the sums
    q = s["q"].double().reshape(r, n, h, -1, dim)
    up, down = q.clamp(min=0).sum(3), q.clamp(max=0).sum(3)                              # [r, n, h, dim]
    b = s["bounds"][s["tables"].long().clamp(min=0)][..., :dim].double()                 # [r, width, h, 2, dim]
    score = torch.einsum("rnhd,rwhd->rnhw", up, b[..., 1, :]) + torch.einsum("rnhd,rwhd->rnhw", down, b[..., 0, :])
    last = (lengths[:, None] - n + torch.arange(n, device="cuda")) // page               # the query's own page
    last = last[:, :, None, None]
    row = torch.arange(width, device="cuda")
    score = score.masked_fill((row < 1) | (row > last - 1), math.inf).masked_fill(row > last, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    best = torch.nn.functional.pad(best, (0, count - best.shape[-1]), value=width)
    best = torch.where(best <= last, best, width).sort(-1).values
    return torch.where(best < width, best, -1).to(torch.int32), s["bounds"]


def _pages_plain(case, s):
    r, n, h, page, dim = (case[x] for x in ("requests", "n", "kv_heads", "page", "dim"))
    pages = s["pages"].long()                                                            # [r, n, h, count]
    entry = torch.gather(s["tables"].long()[:, None, None].expand(r, n, h, -1), 3, pages.clamp(min=0)).clamp(min=0)
    head = torch.arange(h, device="cuda")[:, None]
    k = _values(_nibbles(s["k_codes"][entry, head]), s["k_params"][entry, head], dim).flatten(3, 4)
    v = s["v_codes"][entry, head].transpose(-1, -2).flatten(-3, -2)
    v = _values(_nibbles(v), s["v_params"][entry, head], dim).flatten(3, 4)              # [r, n, h, tokens, dim]
    position = (s["lengths"].long()[:, None] - n + torch.arange(n, device="cuda"))[:, :, None, None, None]
    j = pages[..., None] * page + torch.arange(page, device="cuda")
    mask = ((pages[..., None] >= 0) & (j <= position)).flatten(3, 4)[..., None, :]
    q = s["q"].float().reshape(r, n, h, -1, dim)
    p = _softmax(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim), mask)
    return torch.matmul(p, v).reshape(r, n, case["heads"], dim).to(s["q"].dtype)


def _weigh_plain(case, s):
    r, n, h = case["requests"], case["n"], case["kv_heads"]
    k, v = _tokens(case, s, s["tables"])
    length = s["lengths"].long()[:, None, None]
    position = length - n + torch.arange(n, device="cuda")[None, :, None]
    j = torch.arange(k.shape[-2], device="cuda")
    mask = _rows_mask(case, (j < length) & _sees(position, j, case["window"], case["sinks"]))
    p = _softmax(torch.matmul(_grouped(case, s["q"]), k.transpose(-1, -2)) / math.sqrt(case["dim"]), mask)
    out = _ungrouped(case, torch.matmul(p, v)).to(s["q"].dtype)
    more = p.sum(2).reshape(r, h, -1, case["page"]).transpose(1, 2).flatten(0, 1)        # [r * width, h, page]
    weights = s["weights"].clone()
    return out, weights.index_add_(0, s["tables"].long().clamp(min=0).flatten(), more)


def _evict_plain(case, s):
    weights, lengths, tables, free, count = _restored(s)
    r, h, page, keep, width = case["requests"], case["kv_heads"], case["page"], case["keep"], tables.shape[1]
    cells = width * page
    had = lengths.long()
    over = had > case["limit"]
    at = tables.long().clamp(min=0)
    w = weights[at].transpose(1, 2).reshape(r, h, cells)
    j = torch.arange(cells, device="cuda")
    always = (j < case["first"]) | (j >= had[:, None] - case["last"])
    key = w.masked_fill(always[:, None], math.inf).masked_fill((j >= had[:, None])[:, None], -math.inf)
    best = key.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.nn.functional.pad(best, (0, keep - best.shape[-1]), value=cells)
    best = torch.where(best < had[:, None, None], best, cells).sort(-1).values           # [r, h, keep]
    some = torch.arange(keep, device="cuda") < had[:, None]                              # [r, keep]
    every = torch.where(some, torch.arange(keep, device="cuda"), -1)
    kept = torch.where(over[:, None, None], best, every[:, None])
    # rows of all tokens, [r, h, cells, ...], moved up, and written back to their pages
    moved = torch.where(over[:, None, None], best, torch.arange(keep, device="cuda")).clamp(max=cells - 1)
    token = torch.arange(keep, device="cuda")
    to = torch.gather(at, 1, (token // page).clamp(max=width - 1).expand(r, keep))       # pages of the new places
    write = over[:, None] & (token < cells)
    page_of = torch.where(write, to, at[:, :1])                                          # else the first token, as it is

    def move(name, rows, put):
        x = rows(s[name][at])                                                            # [r, h, cells, c]
        x = torch.gather(x, 2, moved[..., None].expand(-1, -1, -1, x.shape[-1]))
        # places that are not written take their request's first place again, which token 0 has
        x = torch.where(write[:, None, :, None], x, x[:, :, :1])
        put(s[name], x.transpose(1, 2))                                                  # [r, keep, h, c]

    place = torch.where(write, token % page, 0)

    def put_rows(x, y):
        x.transpose(1, 2)[page_of, place] = y

    def put_values(x, y):
        x.permute(0, 2, 4, 1, 3)[page_of, place // 4, place % 4] = y

    def rows(x):
        return x.transpose(1, 2).flatten(2, 3)

    move("k_codes", rows, put_rows)
    move("k_params", rows, put_rows)
    move("v_codes", lambda x: x.transpose(-1, -2).flatten(-3, -2).transpose(1, 2).flatten(2, 3), put_values)
    move("v_params", rows, put_rows)
    # weights of all cells of the requests that lose tokens: the kept ones, zeros behind
    after = torch.zeros_like(w)
    after[..., :keep] = torch.gather(w, 2, moved)[..., :cells]
    after = torch.where(over[:, None, None], after, w)
    own_page = torch.arange(width, device="cuda") < ((had + page - 1) // page)[:, None]  # [r, width]
    pages = free.shape[0]
    weights = torch.cat([weights, weights[:1]])
    weights[torch.where(own_page, at, pages).flatten()] = after.reshape(r, h, width, page).transpose(1, 2).flatten(0, 1)
    weights = weights[:-1]
    # the pages behind, in the order of requests and of their tables, to the end of the free list
    new = torch.where(over, keep, had)
    row = torch.arange(width, device="cuda")
    gone = own_page & (row >= ((new + page - 1) // page)[:, None])
    place = count.long() + torch.cumsum(gone.flatten(), 0) - 1
    free = torch.cat([free, free[:1]])
    free[torch.where(gone.flatten(), place, pages)] = tables.flatten()
    free = free[:-1]
    tables = torch.where(gone, -1, tables)
    count = count + gone.sum().to(torch.int32)
    k, v = _kept_values(case, s)
    i32 = torch.int32
    return kept.to(i32), (had - new).to(i32), new.to(i32), tables, free, count, weights, k, v


def _kept_values(case, s):
    slots, page, dim = s["slots"].long(), case["page"], case["dim"]
    where, off, none = slots.clamp(min=0) // page, slots.clamp(min=0) % page, (slots < 0)[:, None, None]
    k = _values(_nibbles(s["k_codes"].transpose(1, 2)[where, off]), s["k_params"].transpose(1, 2)[where, off], dim)
    v = _nibbles(s["v_codes"].permute(0, 2, 4, 1, 3)[where, off // 4, off % 4])
    return k.masked_fill(none, 0.0), _values(v, s["v_params"].transpose(1, 2)[where, off], dim).masked_fill(none, 0.0)


_PLAIN = {"shared": _shared_plain, "select": _select_plain, "pages": _pages_plain, "weigh": _weigh_plain,
          "evict": _evict_plain}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, h, d, page = case["op"], case["kv_heads"], case["dim"], case["page"]
    held = _held(case)
    row = d / 2 + 4                       # bytes of a key, or of a value
    if op == "evict":
        over = held > case["limit"]
        # every weight is read and written; the kept tokens between first and last are read and written, then read
        kept = np.minimum(held, case["keep"])
        moved = case["keep"] - case["first"]
        return {"bytes": float(h * (8 * held[over].sum() + 2 * 2 * row * moved * over.sum()
                                    + kept.sum() * (2 * row + 8 * d + 4))), "flops": 0}
    size = {"float32": 4}.get(case["dtype"], 2)
    n, heads, group = case["n"], case["heads"], case["heads"] // h
    ends = 2 * size * case["requests"] * n * heads * d
    pairs = keys = 0
    if op == "shared":
        w, prefix, first_seen = case["window"], case["prefix"], case["prefix"]
        for length in held.tolist():
            for i in range(max(0, n - length), n):
                pairs += _visible(prefix + length - n + i, w, case["sinks"])
            if length:
                first = max(0, prefix + length - min(n, length) - w + 1) if w else 0
                keys += length - max(0, first - prefix)
                first_seen = min(first_seen, first)
        keys += prefix - first_seen + min(case["sinks"], first_seen)
        return {"bytes": keys * h * 2 * row + ends, "flops": 4 * pairs * heads * d}
    if op == "select":
        pages = int(-(-held // page).sum())
        fresh = int(np.minimum(case["new"], held).sum())
        return {"bytes": h * (pages * 4 * d + fresh * row) + ends / 2 + 4 * case["requests"] * n * h * case["count"],
                "flops": 4 * pages * n * h * d}
    if op == "pages":
        for length in held.tolist():
            for i in range(n):
                at = length - n + i
                seen = min(case["count"], at // page + 1) * page - (page - 1 - at % page)
                keys += seen
                pairs += seen * group
        return {"bytes": keys * h * 2 * row + ends, "flops": 4 * pairs * h * d}
    w = case["window"]
    for length in held.tolist():
        pairs += sum(_visible(p, w, case["sinks"]) for p in range(length - n, length))
        first = max(0, length - n - w + 1) if w else 0
        keys += length - first + min(case["sinks"], first)
    return {"bytes": keys * h * (2 * row + 8) + ends, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _row64(codes, params, dim):
    digit = torch.arange(codes.shape[-1] * 2, device="cuda")
    byte = codes.long()[..., digit // 2]
    return (((byte >> (4 * (digit % 2))) & 15).double() * params[..., :1].double() + params[..., 1:].double())[..., :dim]


def _held64(case, s, table, tokens):
    """Keys and values of tokens of one request, [tokens, heads, dim]."""
    at, off = table.long()[tokens // case["page"]], tokens % case["page"]
    return (_row64(s["k_codes"][at, :, off], s["k_params"][at, :, off], case["dim"]),
            _row64(s["v_codes"][at, :, off // 4, :, off % 4], s["v_params"][at, :, off], case["dim"]))


def _weights64(q, k, sees):
    """q [h, n, d], k [h, m, d], sees [n, m]: the softmax over what is seen."""
    x = torch.einsum("hnd,hmd->hnm", q, k) / math.sqrt(q.shape[-1])
    x = torch.where(sees, x, torch.full((), -math.inf, dtype=torch.float64, device=x.device))
    return torch.nan_to_num(torch.softmax(x, -1), nan=0.0)


def _sees64(at, m, window, sinks):
    j = torch.arange(m, device="cuda")
    near = torch.ones_like(j <= at[:, None]) if not window else (at[:, None] - j) < window
    return (at[:, None] >= j) & (near | (j < sinks))


def _exact_shared(case, s):
    per, n, prefix, out = case["heads"] // case["kv_heads"], case["n"], case["prefix"], []
    pk, pv = _held64(case, s, s["prefix_table"], torch.arange(prefix, device="cuda"))
    for r, length in enumerate(_held(case).tolist()):
        k, v = _held64(case, s, s["tables"][r], torch.arange(length, device="cuda"))
        k, v = (torch.cat(x).transpose(0, 1) for x in ((pk, k), (pv, v)))
        at = torch.arange(length - n, length, device="cuda")
        sees = _sees64(prefix + at, prefix + length, case["window"], case["sinks"]) & (at >= 0)[:, None]
        o = torch.empty(case["heads"], n, case["dim"], dtype=torch.float64, device="cuda")
        for h in range(case["kv_heads"]):
            q = s["q"][r].double().transpose(0, 1)[h * per:(h + 1) * per]
            o[h * per:(h + 1) * per] = _weights64(q, k[h][None].expand(per, -1, -1), sees) @ v[h]
        out.append(o.transpose(0, 1))
    return torch.stack(out)


def _exact_weigh(case, s):
    per, n, out, weights = case["heads"] // case["kv_heads"], case["n"], [], s["weights"].double()
    for r, length in enumerate(_held(case).tolist()):
        token = torch.arange(length, device="cuda")
        k, v = _held64(case, s, s["tables"][r], token)
        p = _weights64(s["q"][r].double().transpose(0, 1), k.repeat_interleave(per, 1).transpose(0, 1),
                       _sees64(torch.arange(length - n, length, device="cuda"), length, case["window"], case["sinks"]))
        out.append(torch.einsum("hnm,mhd->nhd", p, v.repeat_interleave(per, 1)))
        at, off = s["tables"][r].long()[token // case["page"]], token % case["page"]
        weights[at, :, off] = weights[at, :, off] + p.reshape(-1, per, n, length).sum((1, 2)).T
    return torch.stack(out), weights


def _exact_pages(case, s):
    per, n, page = case["heads"] // case["kv_heads"], case["n"], case["page"]
    held = _held(case).tolist()
    if case["requests"] * n * case["kv_heads"] > 2000:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    pages = s["pages"].cpu()
    for r in range(case["requests"]):
        for i in range(n):
            for h in range(case["kv_heads"]):
                own_pages = pages[r, i, h]
                own_pages = own_pages[own_pages >= 0].long().cuda()
                token = (own_pages[:, None] * page + torch.arange(page, device="cuda")).flatten()
                token = token[token <= held[r] - n + i]
                at, off = s["tables"][r].long()[token // page], token % page
                k = _row64(s["k_codes"][at, h, off], s["k_params"][at, h, off], case["dim"])
                v = _row64(s["v_codes"][at, h, off // 4, :, off % 4], s["v_params"][at, h, off], case["dim"])
                q = s["q"][r, i, h * per:(h + 1) * per].double()
                out[r, i, h * per:(h + 1) * per] = torch.softmax(q @ k.T / math.sqrt(case["dim"]), -1) @ v
    return out


def _exact_select(case, s):
    bounds, page, dim = s["bounds"].double(), case["page"], case["dim"]
    for r, length in enumerate(_held(case).tolist()):
        first = (length - min(case["new"], length)) // page * page
        token = torch.arange(first, length, device="cuda")
        k = _held64(case, s, s["tables"][r], token)[0]
        to = (token - first) // page
        ids = s["tables"][r].long()[first // page:-(-length // page)]
        for side, how in ((0, "amin"), (1, "amax")):
            x = torch.zeros((len(ids), *k.shape[1:]), dtype=torch.float64, device="cuda")
            index = to[:, None, None].expand_as(k)
            bounds[ids, :, side, :dim] = x.scatter_reduce(0, index, k, how, include_self=False)
    return None, bounds


def exact(case, seed):
    one = {"shared": _exact_shared, "weigh": _exact_weigh, "pages": _exact_pages, "select": _exact_select}.get(case["op"])
    # what an eviction leaves are whole numbers and copies of what was held
    return None if one is None else one(case, prepare(case, seed))
