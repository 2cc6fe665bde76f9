"""Serving many requests of different lengths over a paged key/value cache that is held in 8 bits: the four operators
of a step, measured one at a time.

  plan       pages for the new tokens, their positions and the pieces of pages they go to, from request lengths     rai_hip_kv_plan
  rope       rotary positions row by row, and the gradient of it                                      rai_hip_rope_positions
  append     new keys and values into the cache, a power-of-two scale for each page and head                rai_hip_kv_append
  attention  ragged queries over the cache, from one token a request to whole prompts                     rai_hip_kv_attention

The cache is k [pages, kv heads, page, features] and v [pages, kv heads, features, page] in codes of 8 bits ("e4m3", "int8"), and a scale
for each page and head.  Features are the head's, rounded up to a multiple of 16.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": (torch.bfloat16, 2), "f16": (torch.float16, 2), "f32": (torch.float32, 4)}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
FORMAT = {"e4m3": 0, "int8": 1}
E_LEAST, E_MOST = -100, {"e4m3": 119, "int8": 121}


def listed():
    return [
        # One decoding step of 64 requests: the smallest bookkeeping call, latency counts.
        dict(name="plan_decode", kind="plan", requests=64, chunk=1, page=16, table=128, short=False, mix=1),
        # A large batch where prompts are being fed in portions beside decoding requests; long tables.
        dict(name="plan_mixed", kind="plan", requests=512, chunk=160, page=64, table=1024, short=False, mix=2),
        # Queries and keys of a decoding step, a view of the packed projection's rows (Qwen2-1.5B heads).
        dict(name="rope_decode", kind="rope", dtype="bf16", rows=32, heads=14, dim=128, rot=128, interleaved=False, inverse=False, packed=2, far=32768, base=1e6, factor=0.0),
        # Prompts of a Phi-2 batch, two fifths of each head turned.
        dict(name="rope_prompt", kind="rope", dtype="bf16", rows=8192, heads=64, dim=80, rot=32, interleaved=False, inverse=False, packed=32, far=2048, base=1e4, factor=0.0),
        # The gradient for interleaved pairs at far positions of a scaled context, f32.
        dict(name="rope_far_gradient", kind="rope", dtype="f32", rows=4099, heads=16, dim=128, rot=128, interleaved=True, inverse=True, packed=0, far=1000000, base=5e5, factor=8.0),
        # The step's keys and values of 64 requests into pages that are partly full.
        dict(name="append_decode", kind="append", dtype="bf16", format="e4m3", requests=64, chunk=1, context=4096, kv_heads=2, dim=128, page=16, mix=3),
        # Sixteen odd prompts of about a thousand tokens, eight heads.
        dict(name="append_prompts", kind="append", dtype="bf16", format="int8", requests=16, chunk=1300, context=2000, kv_heads=8, dim=128, page=64, mix=4),
        # One request, one token, an odd context: the smallest attention.
        dict(name="attention_one", kind="attention", dtype="bf16", format="e4m3", requests=1, chunk=1, context=777, heads=12, kv_heads=2, dim=128, page=16, window=0, mix=5),
        # A decoding step of 64 requests between 2 k and 16 k tokens.
        dict(name="attention_decode", kind="attention", dtype="bf16", format="e4m3", requests=64, chunk=1, context=16384, heads=12, kv_heads=2, dim=128, page=16, window=0, mix=6),
        # The same for a model with as many key heads as query heads, 80 features (Phi-2), int8, f16 rows.
        dict(name="attention_heads", kind="attention", dtype="f16", format="int8", requests=16, chunk=1, context=2048, heads=32, kv_heads=32, dim=80, page=32, window=0, mix=7),
        # Prompts fed in portions behind what is cached of them.
        dict(name="attention_prompts", kind="attention", dtype="bf16", format="e4m3", requests=4, chunk=1024, context=5000, heads=12, kv_heads=2, dim=128, page=64, window=0, mix=8),
        # Short portions of wide heads (Gemma-2B) in f32 under a sliding window.
        dict(name="attention_window", kind="attention", dtype="f32", format="int8", requests=9, chunk=37, context=2048, heads=8, kv_heads=1, dim=256, page=16, window=512, mix=9),
    ]


def _log(rng, lo, hi):
    """A whole number, even over the logarithm of the range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= 4e10 * (1 if c.get("dtype") != "f32" else 0.25) and w["bytes"] <= 3e8 and _padded(c) <= 3e8:
            return c


def _draw(rng):
    kind, mix = rng.choice(["plan", "rope", "append", "attention", "attention", "attention"]), rng.randrange(1 << 30)
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "plan":
        chunk = rng.choice([1, _log(rng, 2, 1024)])
        return dict(kind=kind, requests=_log(rng, 1, 1024), chunk=chunk, page=page, table=_log(rng, -(-chunk // page) + 1, 2048), short=rng.random() < 0.3, mix=mix)
    dtype, dim = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([64, 72, 80, 128, 128, 256])
    if kind == "rope":
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 8192), heads=_log(rng, 1, 64), dim=dim, rot=rng.choice([dim, dim, 32, 2 * rng.randint(1, dim // 2)]),
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3, packed=rng.choice([0, 1, 8]), far=_log(rng, 1000, 1000000), base=rng.choice([1e4, 5e5, 1e6]),
                    factor=rng.choice([0.0, 8.0]))
    c = dict(kind=kind, dtype=dtype, format=rng.choice(["e4m3", "int8"]), requests=_log(rng, 1, 64), chunk=rng.choice([1, 1, _log(rng, 2, 1500)]))
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    c["context"] = c["chunk"] + _log(rng, 1, 16384) - 1
    if kind == "attention":
        c["heads"] = kv * rng.choice([1, 4, 6, 8]) if kv < 16 else kv
    c.update(kv_heads=kv, dim=dim, page=page, mix=mix)
    if kind == "attention":
        c["window"] = rng.choice([0, 0, _log(rng, 64, 2048)])
    return c


def _padded(case):
    """Keys of a rectangular batch times their size, or their scores: what a plain form unfolds."""
    if "context" not in case:
        return 0
    return case["requests"] * case["context"] * max(case["kv_heads"] * case["dim"], case.get("heads", 0) * case["chunk"])


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """(tokens cached and new, new tokens) of each request, the same for every seed: outputs keep their shapes.  A plan has lengths of its own."""
    rng = random.Random(case["mix"])
    total, new = [], []
    for r in range(case["requests"]):
        n = case["chunk"] if r == 0 or case["chunk"] == 1 else rng.randint(1, case["chunk"])
        if case["kind"] == "plan" and case["chunk"] > 1 and r and rng.random() < 0.6:
            n = rng.choice([0, 1, 1, 1])   # decoding beside the portions of prompts, and requests that pause
        new.append(n)
        if case["kind"] != "plan":
            total.append(case["context"] if r == 0 else _log(rng, max(n, case["context"] // 8), case["context"]))
    return total, new


def _rows_of_runs(n, requests, page):
    return min(n, n // page + 2 * requests)


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def _generator(case, seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 1000003 + 41)


def _features(case):
    return _ceil(case["dim"], 16) * 16


def _frequencies(case):
    """Radians a position, in 64 bits; scaled: waves longer than 8192 positions stretched by the factor, those shorter than
    a quarter of that kept, blended between."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    f = case["base"] ** (-2.0 * i / case["rot"])
    if case["factor"]:
        blend = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        f = (1 - blend) * f / case["factor"] + blend * f
    return f


def _cache(case, g, pages):
    """Keys and values as a model gives them, some features larger than others, in codes and scales."""
    h, d, page = case["kv_heads"], _features(case), case["page"]
    out = {}
    for name, shape, along in (("k", (pages, h, page, d), 3), ("v", (pages, h, d, page), 2)):
        x = torch.randn(shape, generator=g, device="cuda")
        wide = 1 + 3 * (torch.rand(d, generator=g, device="cuda") < 0.05)
        x *= wide.view([-1 if k == along else 1 for k in range(4)])
        if case["dim"] < d:
            x.narrow(along, case["dim"], d - case["dim"]).zero_()
        s = _scale(x.abs().amax((2, 3)), case["format"])
        out[name], out[name + "_scale"] = _codes(x / s[:, :, None, None], case["format"]), s
    return out


def prepare(case, seed):
    g = _generator(case, seed)
    state = dict(case=case)
    kind = case["kind"]
    if kind == "plan":
        R, page, M = case["requests"], case["page"], case["table"]
        _, new = _lengths(case)
        n = sum(new)
        add = torch.tensor(new, dtype=torch.int64, device="cuda")
        lens = ((M * page - add + 1) * torch.rand(R, generator=g, device="cuda", dtype=torch.float64)).long()
        held = (lens + page - 1) // page
        need = int(((lens + add + page - 1) // page - held).sum())
        room = 3 + (need // 2 if case["short"] else need + 5)
        order = torch.randperm(R * M + room, generator=g, device="cuda").to(torch.int32)
        tables = torch.where(torch.arange(M, device="cuda") < held[:, None], order[room:].view(R, M), 0).to(torch.int32)
        free = order[:room]
        taken = torch.full((1,), 3, dtype=torch.int64, device="cuda")
        state.update(lens=lens, add=add, tables=tables, free=free, taken=taken)
        state.update(out_lens=torch.empty_like(lens), out_taken=torch.empty_like(taken), starts=torch.empty(R + 1, dtype=torch.int64, device="cuda"),
                     positions=torch.empty(n, dtype=torch.int64, device="cuda"), runs=torch.empty((4, _rows_of_runs(n, R, page)), dtype=torch.int32, device="cuda"))
        return state
    dt = TYPES[case["dtype"]][0]
    if kind == "rope":
        N, H, D = case["rows"], case["heads"], case["dim"]
        wide = torch.randn((N, H + case["packed"], D), generator=g, device="cuda").to(dt)
        state.update(x=wide[:, :H], positions=torch.randint(0, case["far"], (N,), generator=g, device="cuda"), frequencies=_frequencies(case),
                     magnitude=1.0 + 0.1 * math.log(case["factor"]) if case["factor"] else 1.0, out=torch.empty((N, H, D), dtype=dt, device="cuda"))
        return state
    total, new = _lengths(case)
    R, page, n = case["requests"], case["page"], sum(new)
    M = _ceil(max(total), page)
    pages = sum(_ceil(t, page) for t in total)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    rows, at = [], 0
    for t in total:
        rows.append(order[at:at + _ceil(t, page)] + [0] * (M - _ceil(t, page)))
        at += _ceil(t, page)
    state.update(_cache(case, g, pages))
    if kind == "append":
        runs, at = [], 0
        for r in range(R):
            first = total[r] - new[r]
            for i in range(first // page, _ceil(total[r], page)):
                a, b = max(first, i * page), min(total[r], (i + 1) * page)
                runs.append((rows[r][i], a - i * page, at + a - first, b - a))
            at += new[r]
        state["live"] = len(runs)
        runs += [(0, 0, 0, 0)] * (_rows_of_runs(n, R, page) - len(runs))
        state["runs"] = torch.tensor(runs, dtype=torch.int32, device="cuda").T.contiguous()
        for name in ("new_k", "new_v"):
            state[name] = (torch.randn((n, case["kv_heads"], case["dim"]), generator=g, device="cuda") * 1.1).to(dt)
        return state
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    state.update(tables=torch.tensor(rows, dtype=torch.int32, device="cuda"), starts=torch.tensor(starts, dtype=torch.int64, device="cuda"),
                 lens=torch.tensor(total, dtype=torch.int64, device="cuda"))
    state["q"] = torch.randn((n, case["heads"], case["dim"]), generator=g, device="cuda").to(dt)
    state["out"] = torch.empty_like(state["q"])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    return {"plan": _plan, "rope": _rope, "append": _append, "attention": _attention}[kind](state)


def _results(state):
    kind = state["case"]["kind"]
    if kind == "plan":
        return {k: state[k] for k in ("tables", "out_lens", "out_taken", "starts", "positions", "runs")}
    if kind == "append":
        as_held = torch.float8_e4m3fn if state["case"]["format"] == "e4m3" else torch.int8
        return dict(k=state["k"].view(as_held), v=state["v"].view(as_held), k_scale=state["k_scale"], v_scale=state["v_scale"])
    return state["out"]


def _own(state):
    from rai_amd._lib import call

    c = state["case"]
    d = state.get("descriptors") or _describe(state)   # a program that keeps its tensors keeps their descriptors
    if c["kind"] == "plan":
        call("rai_hip_kv_plan", 0, d["lens"], d["add"], d["free"], d["taken"], d["tables"], c["page"], d["tables"], d["out_lens"], d["out_taken"], d["starts"], d["positions"], d["runs"])
    elif c["kind"] == "rope":
        call("rai_hip_rope_positions", 0, d["x"], d["positions"], d["frequencies"], int(c["interleaved"]), int(c["inverse"]), state["magnitude"], d["out"])
    elif c["kind"] == "append":
        call("rai_hip_kv_append", 0, d["new_k"], d["new_v"], d["runs"], FORMAT[c["format"]], d["k"], d["v"], d["k_scale"], d["v_scale"])
    else:
        call("rai_hip_kv_attention", 0, d["q"], d["tables"], d["starts"], d["lens"], FORMAT[c["format"]], d["k"], d["v"], d["k_scale"], d["v_scale"], c["dim"] ** -0.5, c["window"], d["out"])
    return _results(state)


class _Borrowed:
    """The memory of a torch tensor as a HipTensor's buffer."""

    def __init__(self, t):
        self.t, self.ptr, self.dev = t, t.data_ptr(), 0


def _describe(state):
    from rai_amd._lib import BF16, F16, F32, F64, I64, U8, U32
    from rai_amd.hip import HipTensor

    held = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.float64: F64, torch.int64: I64, torch.int32: U32, torch.uint8: U8}
    state["descriptors"] = {n: HipTensor(_Borrowed(t), held[t.dtype], t.shape, t.stride()).desc() for n, t in state.items() if isinstance(t, torch.Tensor)}
    return state["descriptors"]


# ------------------------------------------------------------------ plain forms
def _plan(state):
    page = state["case"]["page"]
    lens, add, tables, free, taken = (state[k] for k in ("lens", "add", "tables", "free", "taken"))
    R, M = tables.shape
    n, runs = state["positions"].shape[0], state["runs"].shape[1]
    dev = lens.device
    rows = add.clamp(min=0)
    ends = rows.cumsum(0)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), ends])
    fits = (lens >= 0) & (add >= 0) & (lens + add <= M * page) & (ends <= n)
    held = (lens + page - 1) // page
    need = torch.where(fits, (lens + add + page - 1) // page - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= free.shape[0] - taken))
    column = torch.arange(M, device=dev)
    fresh = served[:, None] & (column >= held[:, None]) & (column < (held + need)[:, None])
    source = (taken + (upto - need - held)[:, None] + column).clamp(0, max(free.shape[0] - 1, 0))
    tables.copy_(torch.where(fresh, free[source] if free.shape[0] else 0, tables))
    state["out_lens"].copy_(torch.where(served, lens + add, lens))
    state["out_taken"].copy_(taken + torch.where(served & (need > 0), upto, 0).amax())
    state["starts"].copy_(starts)
    row = torch.arange(n, device=dev)
    r = torch.searchsorted(ends, row, right=True).clamp(max=R - 1)
    state["positions"].copy_(torch.where((row < ends[-1]) & served[r], lens[r] + row - starts[r], -1))
    pieces = torch.where(served & (add > 0), (lens + add - 1) // page - lens // page + 1, 0)
    piece_ends = pieces.cumsum(0)
    w = torch.arange(runs, device=dev)
    r = torch.searchsorted(piece_ends, w, right=True).clamp(max=R - 1)
    i = (lens[r] // page + w - (piece_ends - pieces)[r]).clamp(0, M - 1)
    a, b = torch.maximum(lens[r], i * page), torch.minimum((lens + add)[r], (i + 1) * page)
    pages = tables[r, i].long()
    state["runs"].copy_(torch.where(w < piece_ends[-1], torch.stack([pages, a - i * page, starts[r] + a - lens[r], b - a]), 0))
    return _results(state)


def _rope(state):
    c, x = state["case"], state["x"].float()
    half = c["rot"] // 2
    angle = state["positions"].double()[:, None] * state["frequencies"] * (-1.0 if c["inverse"] else 1.0)
    cos, sin = ((f(angle) * state["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    a, b = (x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) if c["interleaved"] else (x[..., :half], x[..., half:2 * half])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if c["interleaved"] else torch.cat([u, v], -1)
    state["out"].copy_(torch.cat([turned, x[..., c["rot"]:]], -1))
    return _results(state)


def _scale(largest, form):
    """2^e, e the smallest whole number with largest <= LARGEST 2^e."""
    m, e = torch.frexp(largest)
    whole, bits = (0.875, 9) if form == "e4m3" else (127 / 128, 7)
    e = torch.where(largest > 0, e - bits + (m > whole).int(), E_LEAST)
    return torch.ldexp(torch.ones_like(largest), e.clamp(E_LEAST, E_MOST[form]))


def _codes(x, form):
    """Values over their scale as codes, to nearest even; what is not a number as zero."""
    x = torch.where(torch.isnan(x), 0, x).clamp(-LARGEST[form], LARGEST[form])
    return (x.to(torch.float8_e4m3fn) if form == "e4m3" else x.round().to(torch.int8)).view(torch.uint8)


def _values(codes, form):
    return codes.view(torch.float8_e4m3fn if form == "e4m3" else torch.int8).float()


def _append(state):
    c = state["case"]
    form, page = c["format"], c["page"]
    pages, at, row, count = (t[:, None] for t in state["runs"][:, :state["live"]].long())
    j = torch.arange(page, device=at.device) - at
    fresh, before = ((j >= 0) & (j < count))[:, None, :, None], (j < 0)[:, None, :, None]
    source = (row + j).clamp(0, state["new_k"].shape[0] - 1)
    pages = pages[:, 0]
    for name in ("k", "v"):
        x = state["new_" + name][source].float().transpose(1, 2)                       # [run, head, slot, feature]
        x = torch.nn.functional.pad(x, (0, _features(c) - c["dim"]))
        held = state[name][pages]
        held = held if name == "k" else held.transpose(2, 3)
        s_held = state[name + "_scale"][pages]
        s = _scale(torch.where(fresh & torch.isfinite(x), x.abs(), 0).amax((2, 3)), form)
        s = torch.where(at > 0, torch.maximum(s, s_held), s)
        old = _codes(_values(held.contiguous(), form) * (s_held / s)[:, :, None, None], form)
        codes = torch.where(fresh, _codes(x / s[:, :, None, None], form), torch.where(before, old, held))
        state[name][pages] = codes if name == "k" else codes.transpose(2, 3)
        state[name + "_scale"][pages] = s
    return _results(state)


def _attention(state):
    c = state["case"]
    form, R, D, H = c["format"], c["requests"], c["dim"], c["kv_heads"]
    q, tables, starts, lens = state["q"], state["tables"].long(), state["starts"], state["lens"]
    n, group, T = c["chunk"], c["heads"] // H, tables.shape[1] * c["page"]
    at = starts[:-1, None] + torch.arange(n, device=q.device)                          # [request, row]
    k = _values(state["k"][tables], form) * state["k_scale"][tables][..., None, None]     # [request, page, head, slot, feature]
    v = _values(state["v"][tables], form) * state["v_scale"][tables][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(R, H, -1, T)[:, :, :D].contiguous()
    v = v.permute(0, 2, 1, 4, 3).reshape(R, H, T, -1)[..., :D].contiguous()
    rows = q.float()[at.clamp(max=q.shape[0] - 1)].view(R, n, H, group, D).permute(0, 2, 3, 1, 4).reshape(R, H, group * n, D)
    scores = (rows @ k).view(R, H, group, n, T) * (D ** -0.5)
    key, p = torch.arange(T, device=q.device), (lens - starts.diff())[:, None] + torch.arange(n, device=q.device)
    seen = (key <= p[..., None]) & (key < lens[:, None, None])
    if c["window"]:
        seen &= key > p[..., None] - c["window"]
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    out = (w.view(R, H, group * n, T) @ v).view(R, H, group, n, D) / w.sum(-1, keepdim=True).clamp(min=1e-37)
    out = out.permute(0, 3, 1, 2, 4).reshape(R, n, c["heads"], D)
    row = torch.arange(q.shape[0], device=q.device)
    r = torch.searchsorted(starts, row, right=True) - 1
    state["out"].copy_(out[r, row - starts[r]])
    return _results(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "plan":
        R, n, page = case["requests"], sum(_lengths(case)[1]), case["page"]
        return dict(bytes=R * (8 + 8 + 8 + 8) + n * 8 + _rows_of_runs(n, R, page) * 16 + (n // page + R) * 8.0, flops=20.0 * R + 4.0 * n)
    es = TYPES[case["dtype"]][1]
    if case["kind"] == "rope":
        n = case["rows"]
        return dict(bytes=2.0 * n * case["heads"] * case["dim"] * es + 8 * n, flops=3.0 * n * case["heads"] * case["rot"])
    total, new = _lengths(case)
    n, H, D, Dc = sum(new), case["kv_heads"], case["dim"], _features(case)
    if case["kind"] == "append":
        return dict(bytes=2.0 * n * H * (D * es + Dc), flops=6.0 * n * H * D)
    seen = keys = 0
    for t, a in zip(total, new):
        first = t - a
        w = case["window"] or t
        seen += sum(min(p + 1, w) for p in range(first, t))
        keys += t - max(0, first - w + 1)
    return dict(bytes=2.0 * n * case["heads"] * D * es + keys * H * 2.0 * Dc, flops=4.0 * seen * case["heads"] * D)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    if case["kind"] == "plan":
        return None   # whole numbers
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, state)
    if case["kind"] == "append":
        return _exact_append(case, state)
    return _exact_attention(case, state)


def _exact_rope(case, state):
    """Pairs as complex numbers, turned."""
    x, rot = state["x"].double(), case["rot"]
    i = torch.arange(rot // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    z = torch.complex(x[..., first], x[..., second])
    angle = state["positions"].double()[:, None, None] * state["frequencies"]
    z = z * torch.polar(torch.full_like(angle, state["magnitude"]), -angle if case["inverse"] else angle)
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _to_grid(x, form):
    """The nearest value that the format has, the one of the even code where two are as near."""
    if form == "int8":
        return x.round().clamp(-127, 127)
    grid = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64, device=x.device)
    above = torch.searchsorted(grid, x.abs()).clamp(1, 126)
    low, high = grid[above - 1], grid[above]
    up = (x.abs() - low > high - x.abs()) | ((x.abs() - low == high - x.abs()) & (above % 2 == 0))
    return torch.where(up, high, low) * torch.sign(x)


def _exact_append(case, state):
    form, page, d = case["format"], case["page"], case["dim"]
    out = {}
    for name in ("k", "v"):
        codes, scale = _values(state[name], form).double(), state[name + "_scale"].double()
        held = codes if name == "k" else codes.transpose(2, 3)                         # [page, head, slot, feature], a view
        for p, at, row, count in state["runs"][:, :state["live"]].T.tolist():
            x = state["new_" + name][row:row + count].double().transpose(0, 1)
            e = torch.ceil(torch.log2(x.abs().amax((1, 2)) / LARGEST[form])).clamp(E_LEAST, E_MOST[form])
            s = torch.ldexp(torch.ones_like(e), e.int())
            if at:
                s = torch.maximum(s, scale[p])
                held[p, :, :at] = _to_grid(held[p, :, :at] * (scale[p] / s)[:, None, None], form)
            held[p, :, at:at + count, :d] = _to_grid(x / s[:, None, None], form)
            held[p, :, at:at + count, d:] = 0
            scale[p] = s
        out[name], out[name + "_scale"] = (None if form == "int8" else codes), scale
    return out


def _exact_attention(case, state):
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    total, new = _lengths(case)
    group, D, form, row = case["heads"] // case["kv_heads"], case["dim"], case["format"], 0
    for r, (t, a) in enumerate(zip(total, new)):
        pages = state["tables"][r, :_ceil(t, case["page"])].long()
        p = torch.arange(t - a, t, device="cuda")[:, None]
        j = torch.arange(t, device="cuda")[None]
        hidden = (j > p) | ((j <= p - case["window"]) if case["window"] else (j < 0))
        for h in range(case["kv_heads"]):
            k = (_values(state["k"][pages, h], form).double() * state["k_scale"][pages, h].double()[:, None, None]).flatten(0, 1)[:t, :D]
            v = (_values(state["v"][pages, h], form).double() * state["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).flatten(0, 1)[:t, :D]
            for i in range(h * group, (h + 1) * group):
                s = (state["q"][row:row + a, i].double() @ k.T * D ** -0.5).masked_fill(hidden, -math.inf)
                out[row:row + a, i] = torch.softmax(s, 1) @ v
        row += a
    return out
