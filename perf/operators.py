"""Attention over a paged cache of keys and values, as calls of this library's public entry points.

Four operators that a decoder built on the 8-bit fully connected layers runs between them: rotated
queries and appended keys and values (``append``), rows read back from the cache (``gather``), one new
token per sequence against the cache (``decode``) and whole prompts (``prompt``).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes the inputs
and the cache of one, ``run`` is one pass: the library's calls where ``own`` is set, the same operators
from elementary torch operations in 32 bits where it is not. ``exact`` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "s32": torch.int32, "s8": torch.int8}
BASE = 500000.0           # of the rotation's frequencies


# ---- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # one step of eight conversations: the smallest append, all latency
        dict(name="append_b8", op="append", n=8, hq=32, hkv=8, d=128, type="bf16", cache="bf16", page=16,
             heads_first=False, rot=128, interleaved=False, readback=False),
        # a prompt's accumulators straight from the fully connected layers, into an 8-bit cache and back out of it
        dict(name="append_accumulators_4k", op="append", n=4096, hq=32, hkv=8, d=128, type="s32", cache="s8", page=32,
             heads_first=False, rot=128, interleaved=False, readback=True),
        # many packed prompts at once; a head of 80 channels of which 32 are rotated, pairs side by side, pages by head
        dict(name="append_partial_rotation_32k", op="append", n=32768, hq=16, hkv=16, d=80, type="f16", cache="f16",
             page=20, heads_first=True, rot=32, interleaved=True, readback=False),
        # a short shared prefix read back before the rest of its prompt
        dict(name="gather_prefix_333", op="gather", n=333, hkv=8, d=128, type="bf16", cache="s8", page=16,
             heads_first=False),
        # a long document's 8-bit rows read back
        dict(name="gather_document_100k", op="gather", n=100003, hkv=8, d=128, type="bf16", cache="s8", page=64,
             heads_first=True),
        # one conversation, a thousand tokens in: what a single user waits for
        dict(name="decode_b1_1k", op="decode", batch=1, low=1000, high=1000, hq=32, hkv=8, d=128, type="bf16",
             cache="bf16", page=16, heads_first=False, window=0, lse=False),
        # a serving batch of ragged lengths, a few slots empty
        dict(name="decode_b64_ragged_8k", op="decode", batch=64, low=0, high=8192, hq=32, hkv=8, d=128, type="bf16",
             cache="bf16", page=16, heads_first=False, window=0, lse=True),
        # long documents in an 8-bit cache
        dict(name="decode_b8_128k_s8", op="decode", batch=8, low=120000, high=131072, hq=32, hkv=8, d=128,
             type="bf16", cache="s8", page=64, heads_first=True, window=0, lse=False),
        # a head of keys for every head of queries, heads of 80 channels, a sliding window, pages of an odd size
        dict(name="decode_b200_window", op="decode", batch=200, low=1, high=2500, hq=16, hkv=16, d=80, type="f16",
             cache="f16", page=20, heads_first=False, window=1024, lse=False),
        # a chat message
        dict(name="prompt_300", op="prompt", batch=1, low=300, high=300, hq=32, hkv=8, d=128, type="bf16",
             causal=True, window=0, cached=0, pad=0, lse=False),
        # packed prompts of different lengths, the last rows of the buffer unused
        dict(name="prompt_packed_24", op="prompt", batch=24, low=1, high=2048, hq=28, hkv=4, d=64, type="f16",
             causal=True, window=0, cached=0, pad=53, lse=True),
        # a long document
        dict(name="prompt_16k", op="prompt", batch=1, low=16384, high=16384, hq=32, hkv=8, d=128, type="bf16",
             causal=True, window=0, cached=0, pad=0, lse=False),
    ]


HEADS = ((32, 8), (16, 16), (28, 4), (40, 8), (12, 2), (8, 1), (64, 8))
DIMS = (64, 80, 112, 128)
MOST_ELEMENTS = 5e8       # of a drawn cache's keys: half of the largest listed case
MOST_PAIRS = 2e9          # of a drawn prompt's queries and keys, over all heads: a quarter of the largest listed case


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["append", "append", "gather", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    hq, hkv = rng.choice(HEADS)
    d, page, heads_first = rng.choice(DIMS), rng.choice([8, 16, 20, 32, 64, 100]), rng.random() < 0.5
    wide = rng.choice(["f16", "bf16"])
    cache = rng.choice([wide, "s8"])
    if op == "append":
        n = _log(rng, 1, 32768)
        while n * (hq + 2 * hkv) * d > 2e8:
            n = max(1, n // 2)
        return dict(op=op, n=n, hq=hq, hkv=hkv, d=d, type=rng.choice([wide, "s32"]), cache=cache, page=page,
                    heads_first=heads_first, rot=rng.choice([0, 32, d, d]), interleaved=rng.random() < 0.4,
                    readback=cache == "s8")
    if op == "gather":
        return dict(op=op, n=_log(rng, 1, 100000), hkv=hkv, d=d, type=wide, cache=cache, page=page, heads_first=heads_first)
    if op == "decode":
        batch, high = _log(rng, 1, 256), _log(rng, 1, 131072)
        while batch * high * hkv * d > MOST_ELEMENTS:
            if batch > 1 and rng.random() < 0.5:
                batch //= 2
            else:
                high = max(1, high * 2 // 3)
        return dict(op=op, batch=batch, low=rng.choice([0, 1, high // 2, high]), high=high, hq=hq, hkv=hkv, d=d, type=wide,
                    cache=cache, page=page, heads_first=heads_first,
                    window=0 if rng.random() < 0.7 else _log(rng, 1, high), lse=rng.random() < 0.5)
    batch, high = _log(rng, 1, 48), _log(rng, 1, 12000)
    cached = 0 if rng.random() < 0.7 else _log(rng, 1, 3000)
    while batch * high * (high + cached) * hq > MOST_PAIRS:
        if batch > 1 and rng.random() < 0.5:
            batch //= 2
        else:
            high = max(1, high * 2 // 3)
            cached = cached * 3 // 4
    causal = rng.random() < 0.8
    return dict(op=op, batch=batch, low=rng.choice([1, 1 + high // 2, high]), high=high, hq=hq, hkv=hkv, d=d, type=wide,
                causal=causal, window=_log(rng, 1, high) if causal and rng.random() < 0.25 else 0, cached=cached,
                pad=rng.choice([0, 0, 53]), lse=rng.random() < 0.5)


def _lengths(case):
    """The sequences' lengths: the same for every seed, so that the work is known."""
    r = random.Random(case["batch"] * 1000003 + case["high"])
    got = [r.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    got[r.randrange(len(got))] = case["high"]
    return got


def _cached(case):
    """Keys of each sequence that lie before its first query (a prompt whose beginning is there already)."""
    r = random.Random(case["batch"] * 7 + case["cached"])
    return [r.randint(0, case["cached"]) for _ in range(case["batch"])]


# ---- inputs ---------------------------------------------------------------------------------------

class _Maker:
    """Tensors on the GPU, made from the seed alone."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 7919 + 29)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=dtype)

    def s8(self, *shape):
        """Codes of rows whose largest value is near 127."""
        return self.normal(*shape, dtype=torch.float16).mul_(40).clamp_(-127, 127).round_().to(torch.int8)

    def scale(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV).mul_(0.03).add_(0.01)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _cache(m, case, pages, filled):
    """Pages of keys and values, their scales where they are held in 8 bits, and the library's handle of them."""
    shape = (case["hkv"], case["page"]) if case["heads_first"] else (case["page"], case["hkv"])
    eight = case["cache"] == "s8"
    s = {}
    for n in ("k", "v"):
        if not filled:
            s["cache_" + n] = torch.zeros(pages, *shape, case["d"], dtype=TYPES[case["cache"]], device=DEV)
        elif eight:
            s["cache_" + n] = m.s8(pages, *shape, case["d"])
        else:
            s["cache_" + n] = m.normal(pages, *shape, case["d"], dtype=TYPES[case["cache"]])
        s["scale_" + n] = None if not eight else m.scale(pages, *shape) if filled else torch.zeros(pages, *shape, device=DEV)
    s["cache"] = _library().KVCache(s["cache_k"], s["cache_v"], s["scale_k"], s["scale_v"],
                                    heads_first=case["heads_first"]) if own else None
    return s


def _library():
    from __graft_entry__ import load_package
    return load_package().api


def prepare(case, seed):
    m = _Maker(seed)
    op, d, s = case["op"], case["d"], dict(case=case)
    if op in ("append", "gather"):
        n, page = case["n"], case["page"]
        pages = -(-n // page) + 3
        s.update(_cache(m, case, pages, op == "gather"))
        # the tokens of a sequence follow one another within a page, and the pages lie anywhere
        t = torch.arange(n, device=DEV)
        s["slots"] = m.order(pages)[t // page] * page + t % page
    if op == "append":
        s["positions"] = (torch.randint(0, 100000, (1,), generator=m.g, device=DEV) + t).to(torch.int32)
        rot = case["rot"]
        s["freq"] = torch.pow(BASE, -torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot) if rot else None
        for name, heads in (("q", case["hq"]), ("k", case["hkv"]), ("v", case["hkv"])):
            if case["type"] == "s32":
                # sums of a few thousand products of 8-bit values, and the real value of one step of each channel's
                s[name] = m.normal(n, heads, d).mul_(2e5).to(torch.int32)
                s["step_" + name] = torch.rand(heads * d, generator=m.g, device=DEV).add_(0.5).mul_(1e-5)
            else:
                s[name] = m.normal(n, heads, d, dtype=TYPES[case["type"]])
                s["step_" + name] = None
        wide = torch.bfloat16 if case["type"] == "s32" else TYPES[case["type"]]
        s["q_out"] = torch.empty(n, case["hq"], d, dtype=wide, device=DEV)
    if op == "gather" or op == "append" and case["readback"]:
        wide = torch.bfloat16 if case["type"] == "s32" else TYPES[case["type"]]
        s["k_out"], s["v_out"] = (torch.empty(case["n"], case["hkv"], d, dtype=wide, device=DEV) for _ in range(2))
    if op == "decode":
        lengths, page = _lengths(case), case["page"]
        row = -(-max(lengths) // page)
        s.update(_cache(m, case, case["batch"] * row + 1, True))
        s["table"] = m.order(case["batch"] * row + 1)[:case["batch"] * row].view(case["batch"], row).to(torch.int32)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["q"] = m.normal(case["batch"], case["hq"], d, dtype=TYPES[case["type"]])
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["batch"], case["hq"], device=DEV) if case["lse"] else None
    if op == "prompt":
        lengths, before = _lengths(case), _cached(case)
        nq, nk = sum(lengths) + case["pad"], sum(lengths) + sum(before)
        s["most"] = (max(lengths), max(a + b for a, b in zip(lengths, before)))
        s["cu_q"] = torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)
        s["cu_k"] = torch.tensor([0] + [a + b for a, b in zip(lengths, before)], device=DEV).cumsum(0).to(torch.int32)
        s["q"] = m.normal(nq, case["hq"], d, dtype=TYPES[case["type"]])
        s["k"], s["v"] = (m.normal(nk, case["hkv"], d, dtype=TYPES[case["type"]]) for _ in range(2))
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(nq, case["hq"], device=DEV) if case["lse"] else None
    return s


# ---- one pass ---------------------------------------------------------------------------------------

def run(s):
    return dict(append=_append, gather=_gather, decode=_decode, prompt=_prompt)[s["case"]["op"]](s)


def _append(s):
    c = s["case"]
    if own:
        api = _library()
        api.pulpnn_kv_append(s["cache"], s["slots"], s["k"], s["v"], positions=s["positions"], inv_freq=s["freq"],
                             interleaved=c["interleaved"], q=s["q"], q_out=s["q_out"], q_step=s["step_q"],
                             k_step=s["step_k"], v_step=s["step_v"])
        if c["readback"]:
            api.pulpnn_kv_gather(s["cache"], s["slots"], s["k_out"], s["v_out"])
    else:
        x = {n: s[n].float() if s["step_" + n] is None else s[n].float() * s["step_" + n].view(1, -1, c["d"]) for n in "qkv"}
        s["q_out"].copy_(_rotate(x["q"], s, c))
        _store(s, c, "k", _rotate(x["k"], s, c))
        _store(s, c, "v", x["v"])
        if c["readback"]:
            _load_into(s, c)
    if c["readback"]:
        return s["q_out"], s["k_out"], s["v_out"]
    return s["q_out"], s["cache_k"], s["cache_v"]


def _rotate(x, s, c):
    rot = c["rot"]
    if not rot:
        return x
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _slots_first(x, c):
    return x.transpose(1, 2) if c["heads_first"] else x


def _store(s, c, name, x):
    at = s["slots"] // c["page"], s["slots"] % c["page"]
    if c["cache"] == "s8":
        most = x.abs().amax(-1)
        _slots_first(s["scale_" + name], c)[at] = most / 127
        x = (x * (127 / most.clamp(min=1e-30))[..., None]).round()
    _slots_first(s["cache_" + name], c)[at] = x.to(TYPES[c["cache"]])


def _load_into(s, c):
    at = s["slots"] // c["page"], s["slots"] % c["page"]
    for n in "kv":
        x = _slots_first(s["cache_" + n], c)[at].float()
        s[n + "_out"].copy_(x * _slots_first(s["scale_" + n], c)[at][..., None] if c["cache"] == "s8" else x)


def _gather(s):
    if own:
        _library().pulpnn_kv_gather(s["cache"], s["slots"], s["k_out"], s["v_out"])
    else:
        _load_into(s, s["case"])
    return s["k_out"], s["v_out"]


def _softmax(x):
    """Weights and the logarithm of their sum along the last axis; a row of minus infinities has weights of zero."""
    top = x.amax(-1, keepdim=True)
    e = (x - top.clamp(min=-1e30)).exp()
    total = e.sum(-1, keepdim=True)
    return e / total.clamp(min=1e-30), (top + total.log()).squeeze(-1)


def _decode(s):
    c = s["case"]
    if own:
        _library().pulpnn_attn_decode(s["cache"], s["q"], s["table"], s["lengths"], s["out"], window=c["window"], lse=s["lse"])
    else:
        row = torch.arange(s["table"].shape[1] * c["page"], device=DEV)
        pages, at = s["table"].long()[:, row // c["page"]], row % c["page"]
        rows = {n: _slots_first(s["cache_" + n], c)[pages, at].float() for n in "kv"}
        if c["cache"] == "s8":
            for n in "kv":
                rows[n] *= _slots_first(s["scale_" + n], c)[pages, at][..., None]
        q = s["q"].float().view(c["batch"], c["hkv"], -1, c["d"])
        x = torch.einsum("bhgd,bthd->bhgt", q, rows["k"]) / math.sqrt(c["d"])
        n = s["lengths"].long()[:, None]
        seen = (row < n) & (row >= n - c["window"]) if c["window"] else row < n
        w, lse = _softmax(x.masked_fill(~seen[:, None, None], -math.inf))
        s["out"].copy_(torch.einsum("bhgt,bthd->bhgd", w, rows["v"]).reshape(s["out"].shape))
        if s["lse"] is not None:
            s["lse"].copy_(lse.reshape(s["lse"].shape))
    return s["out"] if s["lse"] is None else (s["out"], s["lse"])


def _prompt(s):
    c = s["case"]
    if own:
        _library().pulpnn_attn_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["out"], cu_k=s["cu_k"], causal=c["causal"],
                                      window=c["window"], lse=s["lse"])
    else:
        # every sequence as a row of its own, padded to the longest one
        cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
        i, j = (torch.arange(n, device=DEV) for n in s["most"])
        nq, nk = cu_q.diff()[:, None, None], cu_k.diff()[:, None, None]
        at_q = (cu_q[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
        at_k = (cu_k[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
        seen = (j[None, None] < nk) & (i[None, :, None] < nq)
        last = i[None, :, None] + nk - nq
        if c["causal"]:
            seen = seen & (j <= last)
        if c["window"]:
            seen = seen & (j > last - c["window"])
        token = torch.arange(s["q"].shape[0], device=DEV)
        of = torch.bucketize(token, cu_q[1:], right=True).clamp(max=c["batch"] - 1)
        used, within = token < cu_q[-1], (token - cu_q[of]).clamp(max=s["most"][0] - 1)
        group = c["hq"] // c["hkv"]
        for h in range(c["hkv"]):        # a head of keys at a time: the scores of all of them do not fit the card
            heads = slice(h * group, (h + 1) * group)
            x = torch.einsum("bigd,bjd->bgij", s["q"][:, heads].float()[at_q], s["k"][:, h].float()[at_k]) / math.sqrt(c["d"])
            w, lse = _softmax(x.masked_fill_(~seen[:, None], -math.inf))
            o = torch.einsum("bgij,bjd->bigd", w, s["v"][:, h].float()[at_k])[of, within]
            s["out"][:, heads] = torch.where(used[:, None, None], o.to(s["out"].dtype), s["out"][:, heads])
            if s["lse"] is not None:
                s["lse"][:, heads] = torch.where(used[:, None], lse.transpose(1, 2)[of, within], s["lse"][:, heads])
    return s["out"] if s["lse"] is None else (s["out"], s["lse"])


# ---- what a pass cannot do without ------------------------------------------------------------------

def _size(name):
    return torch.tensor([], dtype=TYPES[name]).element_size()


def work(case):
    op, d = case["op"], case["d"]
    if op in ("append", "gather"):
        n, row = case["n"], 2 * case["hkv"]
        held = n * row * (d * _size(case["cache"]) + (4 if case["cache"] == "s8" else 0))
        if op == "gather":
            return dict(bytes=held + n * row * d * 2 + n * 8, flops=n * row * d)
        both = (case["hq"] + row) * d
        total = n * both * _size(case["type"]) + n * case["hq"] * d * 2 + held + n * 12
        if case["readback"]:
            total += held + n * row * d * 2 + n * 8
        return dict(bytes=total, flops=n * both * 4)
    if op == "decode":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        rows = seen * case["hkv"] * 2 * (d * _size(case["cache"]) + (4 if case["cache"] == "s8" else 0))
        return dict(bytes=rows + case["batch"] * case["hq"] * (d * 4 + (4 if case["lse"] else 0)) + seen // case["page"] * 4,
                    flops=4 * seen * case["hq"] * d)
    pairs = 0
    for a, b in zip(_lengths(case), _cached(case)):
        w = case["window"] or a + b
        if not case["causal"]:
            pairs += a * (a + b)
        else:                            # query i sees min(i + b + 1, w) keys
            short = max(0, min(a, w - b - 1))
            pairs += short * (b + 1) + short * (short - 1) // 2 + (a - short) * min(w, a + b)
    a, b = sum(_lengths(case)), sum(_cached(case))
    return dict(bytes=a * case["hq"] * (d * 4 + (4 if case["lse"] else 0)) + (a + b) * case["hkv"] * d * 4,
                flops=4 * pairs * case["hq"] * d)


# ---- the definitions in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return dict(append=_exact_append, gather=_exact_gather, decode=_exact_decode, prompt=_exact_prompt)[case["op"]](case, s)


def _exact_rows(case, s, name, slots):
    """Rows of the cache as 64-bit values: [slot][head][channel]."""
    x, scale = s["cache_" + name], s["scale_" + name]
    page, at = torch.div(slots, case["page"], rounding_mode="floor"), slots.remainder(case["page"])
    if case["heads_first"]:
        rows = x[page, :, at].double()
        return rows if scale is None else rows * scale[page, :, at].double().unsqueeze(-1)
    rows = x[page, at].double()
    return rows if scale is None else rows * scale[page, at].double().unsqueeze(-1)


def _exact_gather(case, s):
    return tuple(_exact_rows(case, s, n, s["slots"]) for n in ("k", "v"))


def _exact_append(case, s):
    d, rot = case["d"], case["rot"]
    x = {}
    for n in ("q", "k", "v"):
        x[n] = s[n].double()
        if s["step_" + n] is not None:
            x[n] = x[n] * s["step_" + n].double().reshape(-1, d)
    if rot:
        turn = torch.polar(torch.ones(case["n"], rot // 2, dtype=torch.float64, device=DEV),
                           torch.outer(s["positions"].double(), s["freq"]))[:, None]
        for n in ("q", "k"):
            part = x[n][..., :rot]
            pairs = part.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
            pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
            x[n] = torch.cat([pairs.reshape(part.shape), x[n][..., rot:]], -1)
    if case["readback"]:
        held = []
        for n in ("k", "v"):
            step = x[n].abs().amax(-1, keepdim=True) / 127 if case["cache"] == "s8" else None
            held.append(torch.round(x[n] / step) * step if step is not None else x[n])
        return (x["q"], *held)
    if case["cache"] == "s8":
        return x["q"], None, None
    held = []
    for n in ("k", "v"):
        full = s["cache_" + n].double()
        page, at = torch.div(s["slots"], case["page"], rounding_mode="floor"), s["slots"].remainder(case["page"])
        if case["heads_first"]:
            full[page, :, at] = x[n]
        else:
            full[page, at] = x[n]
        held.append(full)
    return (x["q"], *held)


def _exact_attention(q, k, v, seen):
    """One head: its queries [n, d], keys and values [m, d], what each query sees [n, m]."""
    x = (q @ k.T) * q.shape[1] ** -0.5
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, -1)
    w = torch.where(seen, torch.exp(x - lse[:, None]), torch.zeros((), dtype=x.dtype, device=x.device))
    return w @ v, lse


def _exact_decode(case, s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["out"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    group = case["hq"] // case["hkv"]
    for b, n in enumerate(_lengths(case)):
        t = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device=DEV)
        if not len(t):
            continue
        slots = s["table"][b].long()[t // case["page"]] * case["page"] + t % case["page"]
        k, v = (_exact_rows(case, s, x, slots).transpose(0, 1) for x in ("k", "v"))
        q = s["q"][b].double().view(case["hkv"], group, -1)
        x = (q @ k.transpose(1, 2)) * case["d"] ** -0.5
        lse[b] = torch.logsumexp(x, -1).flatten()
        out[b] = (torch.softmax(x, -1) @ v).flatten(0, 1)
    return out if s["lse"] is None else (out, lse)


def _exact_prompt(case, s):
    out, lse = s["out"].double(), torch.zeros(s["out"].shape[:2], dtype=torch.float64, device=DEV)
    group = case["hq"] // case["hkv"]
    q0 = k0 = 0
    for a, b in zip(_lengths(case), _cached(case)):
        i, j = torch.arange(a, device=DEV)[:, None] + b, torch.arange(a + b, device=DEV)
        seen = (j <= i) if case["causal"] else torch.ones(a, a + b, dtype=torch.bool, device=DEV)
        if case["window"]:
            seen = seen & (i - j < case["window"])
        for h in range(case["hq"]):
            k, v = (s[x][k0:k0 + a + b, h // group].double() for x in ("k", "v"))
            out[q0:q0 + a, h], lse[q0:q0 + a, h] = _exact_attention(s["q"][q0:q0 + a, h].double(), k, v, seen)
        q0, k0 = q0 + a, k0 + a + b
    return out if s["lse"] is None else (out, lse)
