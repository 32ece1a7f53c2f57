"""The operators that serve a batch of requests from one 8-bit cache: what they cost, and what they answer.

A serving step is planned on the GPU from the requests' lengths (``kv_block_tables``: pages taken and given back, the slot and
position of every new token), the new keys and values go into the cache (``kv_append_blocks_e4m3_d128``), and all requests
attend to theirs in one dispatch (``attn_blocks_e4m3_d128``).  The cache holds e4m3 numbers in tiles of 16 tokens of one kv head,
each tile with one power of two as its scale; a request's tiles stand in pages named by its row of the block table.

A step whose requests bring one token each is recorded once and replayed, as the lengths are read on the device; the others are
dispatched.  Lengths of a case follow from the case, values from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

D, TILE = 128, 16          # head_dim; tokens of a tile, which share a scale
NONE = -1                  # a slot map's word for "no slot" (0xffffffff)
LOWEST, LARGEST = -15, 61440.0  # least exponent of a tile; largest magnitude that a cache holds


def listed():
    return [
        # The plan of one decode step of 64 conversations: latency alone.
        {"name": "plan_64", "kind": "plan", "requests": 64, "page": 256, "longest": 32768, "tokens": 64, "busy": 0.0, "mix": 1},
        # A step of a large server with small pages: an eighth of the requests has ended, an eighth begins with a prompt.
        {"name": "plan_1024_prompts", "kind": "plan", "requests": 1024, "page": 16, "longest": 4096, "tokens": 16384, "busy": 0.25, "mix": 2},
        # One new token of each of 64 conversations.
        {"name": "append_64", "kind": "append", "requests": 64, "most": 1, "kv": 16, "page": 256, "mix": 3},
        # Prompts of odd lengths, about 16384 tokens in all.
        {"name": "append_prompts", "kind": "append", "requests": 17, "most": 2047, "kv": 16, "page": 64, "mix": 4},
        # One short conversation alone on the GPU: the smallest call.
        {"name": "decode_1_of_1000", "kind": "attend", "requests": 1, "least": 1000, "longest": 1000, "most": 1, "singles": 1.0, "kv": 16, "group": 2,
         "page": 256, "window": 0, "mix": 5},
        # An ordinary decode step: 64 conversations between 256 and 8192 tokens.
        {"name": "decode_64", "kind": "attend", "requests": 64, "least": 256, "longest": 8192, "most": 1, "singles": 1.0, "kv": 16, "group": 2,
         "page": 256, "window": 0, "mix": 6},
        # Many short ones, eight kv heads with four query heads each (a rank's slice of a wider model), small pages.
        {"name": "decode_256_short", "kind": "attend", "requests": 256, "least": 17, "longest": 2048, "most": 1, "singles": 1.0, "kv": 8, "group": 4,
         "page": 16, "window": 0, "mix": 7},
        # One conversation over the longest context that the benchmark quotes.
        {"name": "decode_1_of_131072", "kind": "attend", "requests": 1, "least": 131072, "longest": 131072, "most": 1, "singles": 1.0, "kv": 16, "group": 2,
         "page": 256, "window": 0, "mix": 8},
        # Drafts of four tokens verified in 16 conversations.
        {"name": "verify_16_of_32768", "kind": "attend", "requests": 16, "least": 4000, "longest": 32768, "most": 4, "singles": 0.0, "kv": 16, "group": 2,
         "page": 256, "window": 0, "mix": 9},
        # A sliding layer's decode: of up to 16384 cached tokens the last 1024 count.
        {"name": "decode_32_window", "kind": "attend", "requests": 32, "least": 100, "longest": 16384, "most": 1, "singles": 1.0, "kv": 16, "group": 2,
         "page": 64, "window": 1024, "mix": 10},
        # Prompts and single tokens in one step: three quarters of 24 requests decode, the others bring up to 1500 tokens.
        {"name": "mixed_24", "kind": "attend", "requests": 24, "least": 1, "longest": 4096, "most": 1500, "singles": 0.75, "kv": 16, "group": 2,
         "page": 64, "window": 0, "mix": 11},
        # The last chunk (up to 2048 tokens) of a 64K prompt: the largest call.
        {"name": "chunk_of_65536", "kind": "attend", "requests": 1, "least": 65536, "longest": 65536, "most": 2048, "singles": 0.0, "kv": 16, "group": 2,
         "page": 256, "window": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "attend"])
    page, mix = rng.choice([16, 32, 64, 256, 512]), rng.randint(100, 1 << 20)
    if kind == "plan":
        requests, busy = _log(rng, 1, 4096), rng.choice([0.0, rng.uniform(0.02, 0.5)])
        return {"kind": kind, "requests": requests, "page": page, "longest": _log(rng, 300, 32768 if requests < 500 else 4096),
                "tokens": _log(rng, requests, 32768), "busy": busy, "mix": mix}
    kv = rng.choice([16, 16, 8, 4, 2, 1, 5])
    if kind == "append":
        requests = _log(rng, 1, 512)
        return {"kind": kind, "requests": requests, "most": rng.choice([1, 4, _log(rng, 1, max(1, 32768 // requests))]), "kv": kv, "page": page, "mix": mix}
    group = rng.choice([1, 2, 2, 4, 8])
    form = rng.choice(["decode", "decode", "verify", "prompts"])
    requests = _log(rng, 1, 256 if form != "prompts" else 16)
    longest = _log(rng, 64, min(131072, 2_000_000 // requests))
    most = 1
    if form == "verify":
        most = rng.randint(1, 8)
    if form == "prompts":  # the plain form holds every score of the longest prompt against the longest context
        longest = min(longest, 32768)
        most = min(longest, _log(rng, 16, 4096), max(16, 100_000_000 * 32 // (requests * longest * kv * group)))
    return {"kind": "attend", "requests": requests, "least": rng.choice([most, longest]) if longest > most else longest, "longest": longest, "most": most,
            "singles": rng.choice([0.0, 0.5]) if form == "prompts" else 0.0, "kv": kv, "group": group, "page": page,
            "window": rng.choice([0, 0, 1024, _log(rng, 1, 4096)]), "mix": mix}


# ---- lengths: of the case alone ---------------------------------------------------------------------------------------------
def _attend_lengths(c):
    """(keys, new tokens) of every request, the new tokens among its keys."""
    rng = random.Random(c["mix"])
    keys = [_log(rng, c["least"], c["longest"]) for _ in range(c["requests"])]
    new = [1 if rng.random() < c["singles"] else rng.randint(max(1, c["most"] // 2), c["most"]) for _ in keys]
    return [max(k, n) for k, n in zip(keys, new)], new


def _append_lengths(c):
    """(tokens cached before, new tokens) of every request."""
    rng = random.Random(c["mix"])
    return [rng.randint(0, 3 * c["page"]) for _ in range(c["requests"])], [rng.randint(max(1, c["most"] // 3), c["most"]) for _ in range(c["requests"])]


def _plan_lengths(c):
    """(tokens cached, new tokens, pages held) of every request.  Of the busy ones half have ended, half begin with a prompt."""
    rng = random.Random(c["mix"])
    ctx, new, held = [], [], []
    prompt = max(1, int((c["tokens"] - c["requests"]) / max(1.0, 0.4 * c["busy"] * c["requests"])))
    for _ in range(c["requests"]):
        had = _log(rng, 1, c["longest"] - 1)
        state = rng.random()
        if state < c["busy"] / 2:  # ended: its pages go back
            ctx.append(0), new.append(0), held.append(-(-had // c["page"]))
        elif state < c["busy"]:
            ctx.append(0), new.append(rng.randint(1, min(prompt, c["longest"]))), held.append(0)
        else:
            ctx.append(had), new.append(1), held.append(-(-had // c["page"]))
    return ctx, new, held


# ---- states ----------------------------------------------------------------------------------------------------------------
class _State:
    """Named tensors of one case; what the framework keeps beside them is made by the first pass."""

    def __init__(self, case, seed):
        self.case = case
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        self.t = {}
        self.calls = None
        self.graph = None

    def ints(self, name, values):
        self.t[name] = torch.from_numpy(np.ascontiguousarray(values, dtype=np.int64).astype(np.int32)).cuda()

    def none(self, name, n):
        self.t[name] = torch.full((n,), NONE, dtype=torch.int32, device="cuda")

    def normal(self, name, *shape):
        self.t[name] = torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float16)

    def tables(self, pages, spare):
        """Rows of a block table over a shuffled pool; the entries behind a request's pages are old ones.  The pages left over."""
        stride = max(1, max(pages))
        order = self.rng.permutation(sum(pages) + spare)
        table = self.rng.integers(0, len(order), (len(pages), stride))
        at = 0
        for r, n in enumerate(pages):
            table[r, :n] = order[at:at + n]
            at += n
        self.ints("table", table)
        return order[at:]

    def pool(self, blocks, kv):
        """A cache as appends leave it: a tile's largest magnitude near 448, its exponent the token's and the head's own."""
        for side, lo in (("k", -8), ("v", -9)):
            # e4m3 of N(0, 1) * 100: 4.4 sigma fit, as in a tile of 2048 values; the real values have a deviation of 0.2 to 1.6
            q = (torch.randn(blocks, kv, TILE, D, generator=self.gen, device="cuda", dtype=torch.float16) * 100).clamp_(-448, 448)
            self.t[side + "q"] = q.to(torch.float8_e4m3fn)
            self.t[side + "e"] = torch.randint(lo, -5, (blocks, kv), generator=self.gen, device="cuda", dtype=torch.int8)


def _prepare_plan(s, c):
    ctx, new, held = _plan_lengths(c)
    stride = -(-(c["longest"] + 1) // c["page"])
    order = s.rng.permutation(sum(held) + 2 * c["requests"] + c["tokens"] // c["page"])
    table = s.rng.integers(0, len(order), (len(held), stride))
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    free = np.zeros(len(order), np.int64)
    free[:len(order) - at] = order[at:]
    s.ints("table", table), s.ints("free", free), s.ints("count", [len(order) - at])
    s.ints("ctx", ctx), s.ints("new", new), s.ints("held", held)
    for name, n in (("held_out", len(held)), ("free_out", 4), ("starts", len(held) + 1), ("lens", len(held)), ("slots", c["tokens"]), ("at", c["tokens"])):
        s.none(name, n)


def _prepare_append(s, c):
    ctx, new = _append_lengths(c)
    per = c["page"] // TILE
    pages = [-(-(a + b) // c["page"]) for a, b in zip(ctx, new)]
    s.tables(pages, 1)
    table, slots = s.t["table"].cpu().numpy(), []
    for r, (a, b) in enumerate(zip(ctx, new)):
        pos = np.arange(a, a + b)
        slots.append(table[r, pos // c["page"]].astype(np.int64) * c["page"] + pos % c["page"])
    s.ints("slots", np.concatenate(slots))
    s.pool((sum(pages) + 1) * per, c["kv"])
    n = sum(new)
    s.normal("k", n, c["kv"], D), s.normal("v", n, c["kv"], D)


def _prepare_attend(s, c):
    keys, new = _attend_lengths(c)
    pages = [-(-k // c["page"]) for k in keys]
    s.tables(pages, 1)
    s.pool((sum(pages) + 1) * (c["page"] // TILE), c["kv"])
    s.ints("lens", keys), s.ints("starts", np.concatenate([[0], np.cumsum(new)]))
    s.normal("q", sum(new), c["kv"] * c["group"], D)
    s.t["out"] = torch.zeros(sum(new), c["kv"] * c["group"], D, dtype=torch.float16, device="cuda")


def prepare(case, seed):
    s = _State(case, seed)
    {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend}[case["kind"]](s, case)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------------
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import super_gemma_b200 as sg

        stream = torch.cuda.Stream()
        _ctx = sg.GpuContext(torch.cuda.current_device(), stream=stream.cuda_stream)
        _ctx.stream_object = stream
    return _ctx


def _bound(ctx, s, kernel, names, push, groups):
    import super_gemma_b200 as sg

    at = [s.t[n] for n in names.split()]
    buffers = [ctx.adopt(t.data_ptr(), t.numel() * t.element_size(), np.uint8, keep=t) for t in at]
    return ctx.load_kernel(kernel), [sg.BufferBinding.buffer(i, b) for i, b in enumerate(buffers)], push, groups


def _calls(ctx, s, c):
    if c["kind"] == "plan":
        return _bound(ctx, s, "kv_block_tables", "ctx new held count free table held_out free_out starts lens slots at",
                      (c["page"], s.t["table"].shape[1]), [c["requests"], c["tokens"], 1])
    if c["kind"] == "append":
        return _bound(ctx, s, "kv_append_blocks_e4m3_d128", "k v slots kq ke vq ve", None, [c["kv"], s.t["slots"].numel(), 1])
    tokens = s.t["q"].shape[0]
    work = ctx.attn_blocks_work_bytes(c["kv"], c["group"], c["requests"], tokens, c["most"])
    s.t["work"] = torch.empty(work, dtype=torch.uint8, device="cuda")
    return _bound(ctx, s, "attn_blocks_e4m3_d128", "q kq ke vq ve table lens starts out work",
                  (1.0 / math.sqrt(D), c["page"], s.t["table"].shape[1], c["window"], c["group"], c["most"]), [c["kv"], c["requests"], tokens])


def _run_own(s):
    ctx = _context()
    if s.calls is None:
        s.calls = _calls(ctx, s, s.case)
        if s.case.get("most", 1) == 1 and not s.case.get("busy"):  # one token a request: a step that is recorded and replayed
            s.graph = ctx.record_graph(lambda at: at.dispatch(*s.calls))
    if s.graph is not None:
        ctx.submit(s.graph)
    else:
        ctx.dispatch(*s.calls)


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _plain_plan(s, c):
    t, page, tokens = s.t, c["page"], c["tokens"]
    ctx, new, held, table, count = t["ctx"].long(), t["new"].long(), t["held"].long(), t["table"].long(), t["count"].long()
    n, stride = table.shape
    need = (ctx + new + page - 1) // page
    ends = torch.cumsum(new, 0)
    fits = (need <= stride) & (ends <= tokens)
    given = torch.where(fits, (held - need).clamp(min=0), 0)
    want = torch.where(fits, (need - held).clamp(min=0), 0)
    have = count + given.sum()
    taken = torch.cumsum(want, 0)
    granted = fits & ((want == 0) | (taken <= have))
    column = torch.arange(stride, device="cuda")[None, :]
    # back to the end of the list, in the order of requests and pages; one place more catches what stays
    back = (column >= need[:, None]) & (column < held[:, None]) & fits[:, None]
    place = count + (torch.cumsum(given, 0) - given)[:, None] + column - need[:, None]
    free = torch.cat([t["free"].long(), count])
    free[torch.where(back, place, free.numel() - 1)] = table
    # taken from the end
    out = (column >= held[:, None]) & (column < need[:, None]) & granted[:, None]
    place = have - 1 - ((taken - want)[:, None] + column - held[:, None])
    table = torch.where(out, free[torch.where(out, place, 0)], table)
    used = torch.where(granted, want, 0).sum()
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), ends]).clamp(max=tokens)
    at = torch.arange(tokens, device="cuda")
    r = torch.searchsorted(starts[1:], at, right=True)
    real = r < n
    r = r.clamp(max=n - 1)
    pos = torch.where(real, ctx[r] + at - starts[r], 0)
    has = real & granted[r]
    slot = table[r, (pos // page).clamp(max=stride - 1)] * page + pos % page
    words = torch.stack([(have - used)[0], (~granted).sum(), has.sum(), used])
    return {"table": table.int(), "free": free[:-1].int(), "held_out": torch.where(granted, need, held).int(), "free_out": words.int(), "starts": starts.int(),
            "lens": torch.where(granted, ctx + new, 0).int(), "slots": torch.where(has, slot, NONE).int(), "at": pos.int()}


def _exponent(most):
    """The least e of at least LOWEST with `most` <= 448 * 2^e: most = f * 2^k with f in [0.5, 1), 448 = 0.875 * 2^9."""
    f, k = torch.frexp(most)
    return torch.where(most > 0, k - 9 + (f > 0.875).int(), LOWEST).clamp(min=LOWEST)


def _plain_append_side(x, slots, pool, exps):
    x = x.float().clamp(-LARGEST, LARGEST)
    block, row = slots // TILE, slots % TILE
    blocks, kv = exps.shape
    most = torch.zeros(blocks, kv, device="cuda").index_reduce_(0, block, x.abs().amax(-1), "amax")
    first = torch.full((blocks,), TILE, device="cuda").index_reduce_(0, block, row, "amin")
    old = exps.int()
    e = torch.where((first > 0)[:, None], torch.maximum(_exponent(most), old), _exponent(most))
    e = torch.where((first < TILE)[:, None], e, old)
    # tokens that a grown scale finds in its tile
    grown = (torch.arange(TILE, device="cuda")[None, None, :, None] < first[:, None, None, None]) & (e > old)[:, :, None, None]
    again = (pool.float() * torch.exp2((old - e).float())[:, :, None, None]).to(torch.float8_e4m3fn)
    codes = torch.where(grown, again.view(torch.uint8), pool.view(torch.uint8))
    codes[block, :, row] = (x * torch.exp2(-e[block].float())[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    pool.view(torch.uint8).copy_(codes)
    exps.copy_(e.to(torch.int8))


def _plain_append(s, c):
    slots = s.t["slots"].long()
    _plain_append_side(s.t["k"], slots, s.t["kq"], s.t["ke"])
    _plain_append_side(s.t["v"], slots, s.t["vq"], s.t["ve"])


def _plain_attend(s, c):
    """Every request padded to the longest: all scores, one softmax, one sum."""
    t, kv, g, per = s.t, c["kv"], c["group"], c["page"] // TILE
    lens, starts = t["lens"].long(), t["starts"].long()
    new = starts[1:] - starts[:-1]
    keys, new_most = max(_attend_lengths(c)[0]), c["most"]
    n = lens.numel()
    tile = torch.arange(-(-keys // TILE), device="cuda")
    block = t["table"].long()[:, tile // per] * per + tile % per  # (what stands behind a request's pages is some page's number)

    def values(side):
        x = t[side + "q"][block].float() * torch.exp2(t[side + "e"][block].float())[..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, D)

    i = torch.arange(new_most, device="cuda")
    row = (starts[:-1, None] + i[None, :]).clamp(max=t["q"].shape[0] - 1)
    q = t["q"][row].float().reshape(n, new_most, kv, g, D).permute(0, 2, 1, 3, 4).reshape(n, kv, new_most * g, D)
    scores = torch.matmul(q, values("k").transpose(-1, -2)).mul_(1.0 / math.sqrt(D))
    at = (lens - new)[:, None] + i[None, :]
    key = torch.arange(scores.shape[-1], device="cuda")
    hidden = key[None, None, :] > at[:, :, None]
    if c["window"]:
        hidden |= key[None, None, :] <= at[:, :, None] - c["window"]
    scores.masked_fill_(hidden.repeat_interleave(g, 1)[:, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = scores.sub_(most.clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values("v")) / total
    out = torch.where(total > 0, out, 0.0).reshape(n, kv, new_most, g, D).permute(0, 2, 1, 3, 4).reshape(n, new_most, kv * g, D)
    real = i[None, :] < new[:, None]
    t["out"][row[real]] = out[real].half()


def run(state):
    c = state.case
    if own:
        _run_own(state)
    elif c["kind"] == "plan":
        return _plain_plan(state, c)
    elif c["kind"] == "append":
        _plain_append(state, c)
    else:
        _plain_attend(state, c)
    names = {"plan": "table free held_out free_out starts lens slots at", "append": "kq ke vq ve", "attend": "out"}[c["kind"]]
    return {n: state.t[n] for n in names.split()}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------
def _exact_append(s, x, side):
    """The tiles before their rounding to e4m3, tile by tile as the tokens come."""
    q, e = s.t[side + "q"].double(), s.t[side + "e"].cpu().numpy().astype(np.int64)
    slots = s.t["slots"].cpu().numpy().astype(np.int64)
    x = x.double()
    most = x.abs().amax(-1).cpu().numpy()
    shift = np.zeros_like(e)  # how far the exponent of a tile's old tokens grew
    own_e = np.empty((len(slots), e.shape[1]), np.int64)
    i = 0
    while i < len(slots):
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % TILE:
            j += 1
        b = slots[i] // TILE
        a = np.maximum(most[i:j].max(0), 2.0 ** -30)
        grown = np.maximum(np.ceil(np.log2(a / 448.0) - 1e-12).astype(np.int64), LOWEST)
        if slots[i] % TILE:
            grown = np.maximum(grown, e[b])
            shift[b] = grown - e[b]
            at = int(slots[i] % TILE)
            q[b, :, :at] *= torch.from_numpy(2.0 ** -shift[b].astype(np.float64)).cuda()[:, None, None]
        own_e[i:j] = grown
        i = j
    where = torch.from_numpy(slots).cuda()
    q[where // TILE, :, where % TILE] = x * torch.from_numpy(2.0 ** -own_e.astype(np.float64)).cuda()[:, :, None]
    return q


def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["kind"] == "append":
        return {"kq": _exact_append(s, s.t["k"], "k"), "ke": None, "vq": _exact_append(s, s.t["v"], "v"), "ve": None}
    keys, new = _attend_lengths(c)
    table = s.t["table"].cpu().numpy().astype(np.int64)
    out = torch.zeros(s.t["q"].shape, dtype=torch.float64, device="cuda")
    first, per_tile = 0, c["page"] // TILE
    for r, (n, m) in enumerate(zip(keys, new)):
        tiles = np.arange(-(-n // TILE))
        where = torch.from_numpy(table[r, tiles // per_tile] * per_tile + tiles % per_tile).cuda()
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        seen = key <= pos
        if c["window"]:
            seen &= key > pos - c["window"]
        for h in range(c["kv"]):
            k, v = ((s.t[x + "q"][where, h].double() * torch.pow(2.0, s.t[x + "e"][where, h].double())[:, None, None]).reshape(-1, D)[:n] for x in "kv")
            for j in range(h * c["group"], (h + 1) * c["group"]):
                z = s.t["q"][first:first + m, j].double() @ k.T / math.sqrt(D)
                z[~seen] = -math.inf
                out[first:first + m, j] = torch.softmax(z, -1) @ v
        first += m
    return {"out": out}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def _pairs(n, m, window):
    """(visible pairs, keys that any query sees) of m queries at the end of n keys."""
    if not window or window >= n:
        return m * (n - m) + m * (m + 1) // 2, n
    whole = max(0, min(m, n - window + 1))  # queries that see a full window
    part = m - whole
    return whole * window + part * (n - m) + part * (part + 1) // 2, min(n, window + m - 1)


def work(case):
    c = case
    if c["kind"] == "plan":
        ctx, new, held = _plan_lengths(c)
        need = [-(-(a + b) // c["page"]) for a, b in zip(ctx, new)]
        moved = sum(abs(a - b) for a, b in zip(held, need))
        # lengths and pages read, starts, lengths and pages written; a page's number read and written; a slot and a position a token, read from the table
        return {"bytes": 24 * c["requests"] + 8 * moved + 8 * c["tokens"] + 4 * sum(new), "flops": 0}
    if c["kind"] == "append":
        n = sum(_append_lengths(c)[1])
        return {"bytes": n * (4 + 2 * c["kv"] * D * 3), "flops": n * c["kv"] * D * 2 * 3}
    keys, new = _attend_lengths(c)
    pairs, seen = zip(*(_pairs(n, m, c["window"]) for n, m in zip(keys, new)))
    heads = c["kv"] * c["group"]
    read = sum(seen) * c["kv"] * 2 * (D + 1 / TILE) + sum(4 * -(-n // c["page"]) for n in seen)
    return {"bytes": read + sum(new) * heads * D * 4 + 8 * len(new), "flops": 4 * D * heads * sum(pairs)}
