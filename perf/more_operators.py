"""What stands around the attention of a batched serving step, token by token: what it costs, and what it answers.

All tokens of a step are packed, request by request.  Once a step their positions become rows of cosines and sines
(``rope_cos_sin``).  Per layer the residual stream takes what the last block gave and is normed for the next (``block_norms_*``); queries
and keys of heads without norms of their own are turned by those rows (``rope_qk_f16``); heads of 128 dims with norms go from
the projections to the attention's query and the 8-bit cache in one pass (``qkv_norm_rope_append_blocks_e4m3_d128``).  What the cache
holds comes back as f16 rows with ``kv_read_blocks_e4m3_d128``, for a kernel over linear keys and values or for another tier of memory.

A step of single tokens is recorded once and replayed; prompts are dispatched.  Sizes follow from the case, values from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

D, TILE, NONE = 128, 16, -1  # head_dim of the cache; tokens of a tile, which share an exponent; a slot map's word for "no slot"
EPS = 1e-6
REACH = 11.336               # no value of a normed row of 128 is larger: sqrt(128) and a margin for rounding
LOWEST = -15                 # least exponent of a tile
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # The angles of one decode step of 64 conversations, theta 1e6: latency alone.
        {"name": "angles_64", "kind": "angles", "tokens": 64, "rot": 128, "theta": 1e6, "factor": 1.0, "far": 32768, "replay": True},
        # A step of prompts, 32768 tokens in contexts stretched eightfold, positions up to a million.
        {"name": "angles_32768_far", "kind": "angles", "tokens": 32768, "rot": 128, "theta": 1e4, "factor": 8.0, "far": 1048576, "replay": False},
        # The global heads of the reference (512 dims of which 64 pairs turn) in a decode step of 64.
        {"name": "rotate_64_of_512", "kind": "rotate", "tokens": 64, "head_dim": 512, "rot": 128, "layout": 0, "q_heads": 32, "kv_heads": 4, "packed": False,
         "replay": True},
        # A prompt's queries and keys out of the rows that one projection gave, pairs side by side.
        {"name": "rotate_8192_pairs", "kind": "rotate", "tokens": 8192, "head_dim": 128, "rot": 128, "layout": 2, "q_heads": 32, "kv_heads": 16, "packed": True,
         "replay": False},
        # One new token alone: the smallest call.
        {"name": "pre_attn_1", "kind": "pre", "requests": 1, "most": 1, "pad": 0, "q_heads": 32, "kv_heads": 16, "rot": 128, "layout": 0, "page": 256,
         "packed": False, "mix": 1, "replay": True},
        # One new token of each of 64 conversations, in a step that has room for 72.
        {"name": "pre_attn_64", "kind": "pre", "requests": 64, "most": 1, "pad": 8, "q_heads": 32, "kv_heads": 16, "rot": 128, "layout": 0, "page": 256,
         "packed": False, "mix": 2, "replay": True},
        # Prompts of odd lengths, about 20000 tokens in all, out of packed rows.
        {"name": "pre_attn_prompts", "kind": "pre", "requests": 17, "most": 2047, "pad": 0, "q_heads": 32, "kv_heads": 16, "rot": 128, "layout": 0, "page": 64,
         "packed": True, "mix": 3, "replay": False},
        # Between two blocks of a decode step of 64 at the reference's width: post-norm, residual, the next norm.
        {"name": "norms_64", "kind": "norms", "rows": 64, "hidden": 5376, "residual": "f16", "post": True, "gate": 0, "replay": True},
        # The same for a chunk of 8192 tokens with the residual in 32 bits and a gate for each channel.
        {"name": "norms_8192_f32", "kind": "norms", "rows": 8192, "hidden": 5376, "residual": "f32", "post": True, "gate": 1, "replay": False},
        # Many rows of a narrow model, no norm behind the block, bf16, a gate for each token.
        {"name": "norms_30011_bf16", "kind": "norms", "rows": 30011, "hidden": 1096, "residual": "bf16", "post": False, "gate": 2, "replay": False},
        # One short conversation read back.
        {"name": "read_1000", "kind": "read", "requests": 1, "least": 1000, "longest": 1000, "kv_heads": 16, "page": 256, "mix": 4, "replay": False},
        # 40 conversations of odd lengths, small pages, up to 131072 tokens: the largest call.
        {"name": "read_40", "kind": "read", "requests": 40, "least": 300, "longest": 8191, "kv_heads": 16, "page": 16, "mix": 5, "replay": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["angles", "rotate", "rotate", "pre", "pre", "pre", "norms", "norms", "norms", "read", "read"])
    if kind == "angles":
        tokens, rot = _log(rng, 1, 65536), 16 * _log(rng, 1, 32)
        tokens = min(tokens, 8_000_000 // rot)
        return {"kind": kind, "tokens": tokens, "rot": rot, "theta": rng.choice([1e4, 1e6, 5e5]), "factor": rng.choice([1.0, 2.0, 8.0, 32.0]),
                "far": _log(rng, 100, 1 << 24), "replay": tokens <= 512}
    if kind == "rotate":
        head_dim = rng.choice([64, 80, 96, 128, 128, 256, 512, 16 * rng.randint(1, 40)])
        rot = rng.choice([head_dim, 16 * rng.randint(1, head_dim // 16)])
        kv = rng.choice([1, 2, 4, 8, 16, 5])
        heads = kv * rng.choice([1, 2, 4, 7, 8])
        tokens = _log(rng, 1, min(32768, 50_000_000 // (head_dim * (heads + kv))))
        return {"kind": kind, "tokens": tokens, "head_dim": head_dim, "rot": rot, "layout": rng.choice([0, 1, 2]), "q_heads": heads, "kv_heads": kv,
                "packed": rng.random() < 0.5, "replay": tokens <= 512}
    page, mix = rng.choice([16, 32, 64, 256, 512]), rng.randint(100, 1 << 20)
    if kind == "pre":
        kv = rng.choice([16, 16, 8, 4, 2, 1, 5])
        heads = kv * rng.choice([1, 2, 2, 4, 8])
        requests = _log(rng, 1, 512)
        most = rng.choice([1, 4, _log(rng, 1, max(1, min(8192, 170_000_000 // (D * (heads + 2 * kv) * requests))))])
        return {"kind": kind, "requests": requests, "most": most, "pad": rng.choice([0, 0, rng.randint(1, 100)]), "q_heads": heads, "kv_heads": kv,
                "rot": rng.choice([128, 128, 64, 16 * rng.randint(1, 8)]), "layout": rng.choice([0, 0, 1, 2]), "page": page, "packed": rng.random() < 0.5,
                "mix": mix, "replay": requests * most <= 512}
    if kind == "norms":
        hidden = 8 * _log(rng, 1, 2048)
        rows = _log(rng, 1, min(65536, 40_000_000 // hidden))
        return {"kind": kind, "rows": rows, "hidden": hidden, "residual": rng.choice(["f16", "bf16", "f32"]), "post": rng.random() < 0.7,
                "gate": rng.choice([0, 1, 2, 3]), "replay": rows <= 512}
    requests = _log(rng, 1, 300)
    longest = _log(rng, 1, 131072 // requests)
    return {"kind": kind, "requests": requests, "least": rng.randint(1, longest), "longest": longest, "kv_heads": rng.choice([16, 16, 8, 4, 2, 1, 5]),
            "page": page, "mix": mix, "replay": False}


# ---- lengths: of the case alone ---------------------------------------------------------------------------------------------
def _pre_lengths(c):
    """(tokens cached before, new tokens) of every request."""
    rng = random.Random(c["mix"])
    return [rng.randint(0, 3 * c["page"]) for _ in range(c["requests"])], [rng.randint(max(1, c["most"] // 3), c["most"]) for _ in range(c["requests"])]


def _read_lengths(c):
    """(first token, tokens) that are read of every request: half of them from their beginning."""
    rng = random.Random(c["mix"])
    n = [_log(rng, c["least"], c["longest"]) for _ in range(c["requests"])]
    return [rng.choice([0, rng.randint(0, 2 * c["page"])]) for _ in n], n


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

    def normal(self, *shape, dtype=torch.float16, by=1.0):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float32).mul_(by).to(dtype)

    def parts(self, tokens, **widths):
        """Tensors [tokens, width]: of their own, or side by side in one row, as one projection gives them."""
        if not self.case["packed"]:
            for name, w in widths.items():
                self.t[name] = self.normal(tokens, w)
            return
        whole, at = self.normal(tokens, sum(widths.values())), 0
        for name, w in widths.items():
            self.t[name] = whole[:, at:at + w]
            at += w

    def rows(self, tokens, rot, far):
        """Cosines and sines of the tokens' positions."""
        at = torch.from_numpy(self.rng.integers(0, far, tokens)).cuda()
        angle = at.double()[:, None] * torch.from_numpy(_frequencies(rot, 1e6, 1.0)).cuda()[None, :]
        self.t["cos_sin"] = torch.stack([angle.cos(), angle.sin()], -1).float()

    def tables(self, pages, spare):
        """Rows of a block table over a shuffled pool; the entries behind a request's pages are old ones."""
        stride = max(1, max(pages))
        order = self.rng.permutation(sum(pages) + spare)
        table = self.rng.integers(0, len(order), (len(pages), stride))
        at = 0
        for r, n in enumerate(pages):
            table[r, :n] = order[at:at + n]
            at += n
        self.ints("table", table)
        return table

    def pool(self, blocks, kv, k_exp, v_exp):
        """A cache as appends leave it: exponents that the norms' bounds give, one tile of eight as the append of unnormed rows leaves it."""
        for side, e in (("k", k_exp), ("v", v_exp)):
            other = torch.randint(0, 8, (blocks, kv), generator=self.gen, device="cuda") == 0
            by = torch.where(other, 1.0, 0.25)[:, :, None, None]
            q = (self.normal(blocks, kv, TILE, D, by=100.0) * by).clamp_(-448, 448)
            self.t[side + "q"] = q.to(torch.float8_e4m3fn)
            found = torch.randint(-8, -4, (blocks, kv), generator=self.gen, device="cuda")
            self.t[side + "e"] = torch.where(other, found, e).to(torch.int8)


def _frequencies(rot, theta, factor):
    """Radians a position of every pair, 64 bits; for stretched contexts those that turn less than 32 times over 4096 tokens are slowed
    down, by up to `factor` for those that turn once or less."""
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    keep = np.clip((4096 * f / (2 * np.pi) - 1.0) / 31.0, 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep)


def _magnitude(factor):
    return float(np.float32(0.1 * math.log(factor) + 1.0))


def _prepare_angles(s, c):
    s.t["freqs"] = torch.from_numpy(_frequencies(c["rot"], c["theta"], c["factor"])).cuda()
    s.ints("positions", s.rng.integers(0, c["far"], c["tokens"]))
    s.t["cos_sin"] = torch.zeros(c["tokens"], c["rot"] // 2, 2, device="cuda")


def _prepare_rotate(s, c):
    n, d = c["tokens"], c["head_dim"]
    s.parts(n, q=c["q_heads"] * d, k=c["kv_heads"] * d)
    s.rows(n, c["rot"], 32768)
    for x in "qk":
        s.t[x + "_out"] = torch.zeros(s.t[x].shape, dtype=torch.float16, device="cuda")


def _prepare_pre(s, c):
    ctx, new = _pre_lengths(c)
    kv, n = c["kv_heads"], sum(new) + c["pad"]
    s.parts(n, q=c["q_heads"] * D, k=kv * D, v=kv * D)
    s.rows(n, c["rot"], 32768)
    for w in ("q_w", "k_w"):
        s.t[w] = 1.0 + s.normal(D, dtype=torch.float32, by=0.2)
    pages = [-(-(a + b) // c["page"]) for a, b in zip(ctx, new)]
    table, slots = s.tables(pages, 1), []
    for r, (a, b) in enumerate(zip(ctx, new)):
        pos = np.arange(a, a + b)
        slots.append(table[r, pos // c["page"]].astype(np.int64) * c["page"] + pos % c["page"])
    s.ints("slots", np.concatenate(slots + [np.full(c["pad"], NONE)]))
    s.pool((sum(pages) + 1) * (c["page"] // TILE), kv, _exponent((s.t["k_w"].abs().amax() * REACH).clamp(max=61440.0)), -5)
    s.t["q_out"] = torch.zeros(n, c["q_heads"] * D, dtype=torch.float16, device="cuda")


def _prepare_norms(s, c):
    n, h = c["rows"], c["hidden"]
    s.t["y"] = s.normal(n, h)
    s.t["h"] = s.normal(n, h, dtype=TYPES[c["residual"]], by=8.0)
    s.t["w_post"], s.t["w_pre"] = (1.0 + s.normal(h, dtype=torch.float32, by=0.2) for _ in range(2))
    s.t["gate"] = torch.rand((1, h, n, 1)[c["gate"]], generator=s.gen, device="cuda")
    s.t["h_out"] = torch.zeros(n, h, dtype=TYPES[c["residual"]], device="cuda")
    s.t["x"] = torch.zeros(n, h, dtype=torch.float16, device="cuda")


def _prepare_read(s, c):
    first, n = _read_lengths(c)
    pages = [-(-(a + b) // c["page"]) for a, b in zip(first, n)]
    s.tables(pages, 1)
    s.pool((sum(pages) + 1) * (c["page"] // TILE), c["kv_heads"], -5, -5)
    s.ints("first", first), s.ints("starts", np.concatenate([[0], np.cumsum(n)]))
    for x in "kv":
        s.t[x] = torch.zeros(sum(n), c["kv_heads"], D, dtype=torch.float16, device="cuda")


def prepare(case, seed):
    s = _State(case, seed)
    {"angles": _prepare_angles, "rotate": _prepare_rotate, "pre": _prepare_pre, "norms": _prepare_norms, "read": _prepare_read}[case["kind"]](s, case)
    torch.cuda.synchronize()
    return s


SCALE = 0.75  # of the residual stream behind a block


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
    spans = [((t.shape[0] - 1) * t.stride(0) + t[0].numel()) * t.element_size() for t in at]  # a view's rows reach that far
    buffers = [ctx.adopt(t.data_ptr(), n, np.uint8, keep=t) for t, n in zip(at, spans)]
    return ctx.load_kernel(kernel), [sg.BufferBinding.buffer(i, b) for i, b in enumerate(buffers)], push, groups


def _calls(ctx, s, c):
    stride = lambda x: s.t[x].stride(0)  # noqa: E731
    if c["kind"] == "angles":
        return _bound(ctx, s, "rope_cos_sin", "freqs positions cos_sin", (c["rot"], _magnitude(c["factor"])), [c["tokens"], 1, 1])
    if c["kind"] == "rotate":
        return _bound(ctx, s, "rope_qk_f16", "q k cos_sin q_out k_out",
                      (c["head_dim"], c["rot"], c["layout"], stride("q"), stride("k"), stride("q_out"), stride("k_out")), [c["q_heads"], c["kv_heads"], c["tokens"]])
    if c["kind"] == "pre":
        return _bound(ctx, s, "qkv_norm_rope_append_blocks_e4m3_d128", "q q_w q_out k v k_w cos_sin slots kq ke vq ve",
                      (c["rot"], c["layout"], 0, stride("q"), stride("k"), stride("v"), 1.0), [c["q_heads"], c["kv_heads"], s.t["q"].shape[0]])
    if c["kind"] == "norms":
        return _bound(ctx, s, "block_norms_" + c["residual"], "y h w_post gate w_pre h_out x", (1 if c["post"] else 0, c["gate"], 0, SCALE, EPS),
                      [c["hidden"], c["rows"], 1])
    return _bound(ctx, s, "kv_read_blocks_e4m3_d128", "kq ke vq ve table first starts k v", (c["page"], s.t["table"].shape[1]),
                  [c["kv_heads"], c["requests"], s.t["k"].shape[0]])


def _run_own(s):
    ctx = _context()
    if s.calls is None:
        s.calls = _calls(ctx, s, s.case)
        if s.case["replay"]:
            s.graph = ctx.record_graph(lambda at: at.dispatch(*s.calls))
    if s.graph is not None:
        ctx.submit(s.graph)
    else:
        ctx.dispatch(*s.calls)


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _plain_angles(s, c):
    angle = s.t["positions"].double()[:, None] * s.t["freqs"][None, :]  # a far position's angle has no digits left in 32 bits
    s.t["cos_sin"].copy_(torch.stack([angle.cos(), angle.sin()], -1) * _magnitude(c["factor"]))


def _turn(x, cos_sin, layout):
    """x f32 [tokens, heads, dims] turned by the tokens' rows [tokens, pairs, 2]; dims beyond the pairs stay."""
    pairs, half = cos_sin.shape[1], x.shape[2] // 2
    c, sn = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    lo, hi = {0: (slice(0, pairs), slice(half, half + pairs)), 1: (slice(0, pairs), slice(pairs, 2 * pairs)),
              2: (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))}[layout]
    out = x.clone()
    out[:, :, lo] = x[:, :, lo] * c - x[:, :, hi] * sn
    out[:, :, hi] = x[:, :, hi] * c + x[:, :, lo] * sn
    return out


def _plain_rotate(s, c):
    n = c["tokens"]
    for x in "qk":
        s.t[x + "_out"].copy_(_turn(s.t[x].float().reshape(n, -1, c["head_dim"]), s.t["cos_sin"], c["layout"]).reshape(n, -1))


def _normed(x, w):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w


def _exponent(most):
    """The least e of at least LOWEST with `most` <= 448 * 2^e: most = f * 2^k with f in [0.5, 1), 448 = 0.875 * 2^9."""
    f, k = torch.frexp(most)
    return (k - 9 + (f > 0.875).int()).clamp(min=LOWEST)


def _plain_append(x, slots, pool, exps, e):
    """Rows x [n, kv, 128] into their slots; e: the exponent that holds every normed row."""
    block, row = slots // TILE, slots % TILE
    first = torch.full((exps.shape[0],), TILE, device="cuda").index_reduce_(0, block, row, "amin")[:, None]
    old = exps.int()
    new = torch.where(first > 0, torch.maximum(old, e), e.expand_as(old))
    new = torch.where(first < TILE, new, old)
    # tokens that a grown exponent finds in its tile
    grown = (torch.arange(TILE, device="cuda")[None, None, :, None] < first[:, :, None, None]) & (new > old)[:, :, None, None]
    again = (pool.float() * torch.exp2((old - new).float())[:, :, None, None]).to(torch.float8_e4m3fn)
    codes = torch.where(grown, again.view(torch.uint8), pool.view(torch.uint8))
    most = torch.minimum(torch.tensor(448.0, device="cuda"), 61440.0 * torch.exp2(-new.float()))[block, :, None]
    x = x * torch.exp2(-new[block].float())[:, :, None]
    codes[block, :, row] = torch.minimum(torch.maximum(x, -most), most).to(torch.float8_e4m3fn).view(torch.uint8)
    pool.view(torch.uint8).copy_(codes)
    exps.copy_(new.to(torch.int8))


def _plain_pre(s, c):
    t = s.t
    here = t["slots"] != NONE
    slots, n = t["slots"][here].long(), t["slots"].shape[0]
    rows = lambda x: t[x].reshape(n, -1, D)[here].float()  # noqa: E731
    cos_sin = t["cos_sin"][here]
    t["q_out"][here] = _turn(_normed(rows("q"), t["q_w"]), cos_sin, c["layout"]).half().reshape(slots.shape[0], -1)
    bound = (t["k_w"].abs().amax() * REACH).clamp(max=61440.0)
    _plain_append(_turn(_normed(rows("k"), t["k_w"]), cos_sin, c["layout"]), slots, t["kq"], t["ke"], _exponent(bound))
    _plain_append(_normed(rows("v"), None), slots, t["vq"], t["ve"], _exponent(torch.tensor(REACH, device="cuda")))


def _plain_norms(s, c):
    t = s.t
    y = t["y"].float()
    if c["post"]:
        y = _normed(y, t["w_post"])
    if c["gate"]:
        y = y * (t["gate"][:, None] if c["gate"] == 2 else t["gate"])
    h = (t["h"].float() + y) * SCALE
    t["h_out"].copy_(h)
    t["x"].copy_(_normed(h, t["w_pre"]))


def _plain_read(s, c):
    t, page = s.t, c["page"]
    starts = t["starts"].long()
    i = torch.arange(t["k"].shape[0], device="cuda")
    r = torch.searchsorted(starts[1:], i, right=True)
    pos = t["first"].long()[r] + i - starts[r]
    row = t["table"].long()[r, pos // page] * page + pos % page
    for x in "kv":
        q = t[x + "q"][row // TILE, :, row % TILE].float()
        t[x].copy_(q * torch.exp2(t[x + "e"][row // TILE].float())[:, :, None])


PLAIN = {"angles": _plain_angles, "rotate": _plain_rotate, "pre": _plain_pre, "norms": _plain_norms, "read": _plain_read}
OUTPUTS = {"angles": "cos_sin", "rotate": "q_out k_out", "pre": "q_out kq ke vq ve", "norms": "h_out x", "read": "k v"}


def run(state):
    kind = state.case["kind"]
    if own:
        _run_own(state)
    else:
        PLAIN[kind](state, state.case)
    return {n: state.t[n] for n in OUTPUTS[kind].split()}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------
def _exact_turn(x, cos_sin, layout):
    """Pairs as complex numbers times e^(i angle)."""
    pairs, d = cos_sin.shape[1], x.shape[-1]
    i = torch.arange(pairs, device="cuda")
    a, b = (2 * i, 2 * i + 1) if layout == 2 else (i, i + (d // 2 if layout == 0 else pairs))
    z = torch.complex(x[..., a], x[..., b]) * torch.view_as_complex(cos_sin.double().contiguous())[:, None, :]
    out = x.clone()
    out[..., a], out[..., b] = z.real, z.imag
    return out


def _exact_norm(x, w=None):
    y = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS)
    return y if w is None else y * w.double()


def _exact_append(s, x, slots, side, e):
    """The tiles before their rounding to e4m3, tile by tile as the tokens come."""
    q, exps = s.t[side + "q"].double(), s.t[side + "e"].cpu().numpy().astype(np.int64)
    used = np.empty((len(slots), exps.shape[1]), np.int64)
    i = 0
    while i < len(slots):
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % TILE:
            j += 1
        b, at = slots[i] // TILE, int(slots[i] % TILE)
        used[i:j] = e if at == 0 else np.maximum(e, exps[b])
        if at:
            q[b, :, :at] *= torch.from_numpy(2.0 ** (exps[b] - used[i]).astype(np.float64)).cuda()[:, None, None]
        i = j
    where = torch.from_numpy(slots).cuda()
    q[where // TILE, :, where % TILE] = x * torch.from_numpy(2.0 ** -used.astype(np.float64)).cuda()[:, :, None]
    return q


def _exact_read(s, c, side):
    table, per = s.t["table"].cpu().numpy().astype(np.int64), c["page"] // TILE
    out, at = torch.empty(s.t[side].shape, dtype=torch.float64, device="cuda"), 0
    for r, (a, n) in enumerate(zip(*_read_lengths(c))):
        tiles = np.arange(a // TILE, -(-(a + n) // TILE))
        where = torch.from_numpy(table[r, tiles // per] * per + tiles % per).cuda()
        x = s.t[side + "q"][where].double() * torch.pow(2.0, s.t[side + "e"][where].double())[:, :, None, None]
        out[at:at + n] = x.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], D)[a % TILE:a % TILE + n]
        at += n
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    t = s.t
    if c["kind"] == "angles":
        turns = t["positions"].double()[:, None] * t["freqs"]
        return {"cos_sin": torch.view_as_real(torch.polar(torch.full_like(turns, _magnitude(c["factor"])), turns))}
    if c["kind"] == "rotate":
        n, d = c["tokens"], c["head_dim"]
        return {x + "_out": _exact_turn(t[x].double().reshape(n, -1, d), t["cos_sin"], c["layout"]).reshape(n, -1) for x in "qk"}
    if c["kind"] == "pre":
        real, n = sum(_pre_lengths(c)[1]), t["slots"].shape[0]
        slots, cos_sin = t["slots"][:real].cpu().numpy().astype(np.int64), t["cos_sin"][:real]
        rows = lambda x: t[x].reshape(n, -1, D)[:real].double()  # noqa: E731
        q = torch.zeros(n, c["q_heads"] * D, dtype=torch.float64, device="cuda")
        q[:real] = _exact_turn(_exact_norm(rows("q"), t["q_w"]), cos_sin, c["layout"]).reshape(real, -1)
        most = float(np.float32(t["k_w"].abs().max().item()) * np.float32(REACH))
        e = max(LOWEST, math.ceil(math.log2(most / 448.0) - 1e-12))
        k = _exact_append(s, _exact_turn(_exact_norm(rows("k"), t["k_w"]), cos_sin, c["layout"]), slots, "k", e)
        return {"q_out": q, "kq": k, "ke": None, "vq": _exact_append(s, _exact_norm(rows("v")), slots, "v", -5), "ve": None}
    if c["kind"] == "norms":
        n = _exact_norm(t["y"].double(), t["w_post"]) if c["post"] else t["y"].double()
        g = (1.0, t["gate"].double(), t["gate"].double()[:, None], t["gate"].double())[c["gate"]]
        h = (t["h"].double() + g * n) * SCALE
        return {"h_out": h, "x": _exact_norm(h, t["w_pre"])}
    return {x: _exact_read(s, c, x) for x in "kv"}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "angles":
        return {"bytes": c["tokens"] * (4 + 4 * c["rot"]) + 4 * c["rot"], "flops": c["tokens"] * c["rot"]}
    if c["kind"] == "rotate":
        heads = c["q_heads"] + c["kv_heads"]
        return {"bytes": c["tokens"] * (4 * heads * c["head_dim"] + 4 * c["rot"]), "flops": c["tokens"] * heads * c["rot"] * 3}
    if c["kind"] == "pre":
        new, pad = sum(_pre_lengths(c)[1]), c["pad"]
        heads, kv = c["q_heads"], c["kv_heads"]
        return {"bytes": new * (4 * heads * D + 6 * kv * D + 4 * c["rot"]) + 4 * (new + pad), "flops": new * D * (7 * heads + 14 * kv)}
    if c["kind"] == "norms":
        size = TYPES[c["residual"]].itemsize
        vectors = (2 if c["post"] else 1) + (1 if c["gate"] == 1 else 0)
        return {"bytes": c["rows"] * c["hidden"] * (4 + 2 * size) + 4 * c["hidden"] * vectors + (4 * c["rows"] if c["gate"] == 2 else 0),
                "flops": c["rows"] * c["hidden"] * 9}
    n = sum(_read_lengths(c)[1])
    return {"bytes": n * c["kv_heads"] * 6 * D, "flops": n * c["kv_heads"] * 2 * D}
