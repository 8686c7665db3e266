"""Timed calls of positions in attention: what is run, on which inputs, their plain forms and exact values.

What lies between a layer's projection and its attention, and attention whose scores know of positions:

- ``rotate``: rotary positions of queries or keys, whole heads or a part of each, pairs of halves or of neighbours,
  frequencies as they are or scaled for long contexts;
- ``norm``: the norm of every head of queries and keys, and the rotation behind it;
- ``append``: a step's new tokens on their way into a paged cache: keys normed and rotated, values as they are, the
  queries made ready beside them; then the tokens as the cache holds them, read back;
- ``prompt``: attention over packed sequences whose scores are capped, get a bias by distance, or both; in both
  directions, causal, or causal behind a prefix that all see;
- ``step``: attention of each sequence's newest tokens over a paged cache with such scores.

Where ``own`` is false the operators run in their plain form: elementary torch operations in 32 bits, angles in 64.
"""
from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

EPS = 1e-6


def _package():
    name = "cuvs_silicon_amd"
    if name not in sys.modules:
        pkg = os.path.join(ROOT, "cuvs-silicon_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


_ctx = None


def _context():
    """One context for the process, on the stream that the program's tensors are made on."""
    global _ctx
    if _ctx is None:
        _ctx = _package().Context(0, stream=torch.cuda.current_stream().cuda_stream)
    return _ctx


# ---- cases -----------------------------------------------------------------


def _rotate(name, tokens, first, heads, dim, dims, interleaved, scaling, dtype):
    return dict(name=name, kind="rotate", tokens=tokens, first=first, heads=heads, dim=dim, dims=dims,
                interleaved=interleaved, scaling=scaling, dtype=dtype)


def _norm(name, tokens, first, heads, kv_heads, dim, dims, interleaved, dtype):
    return dict(name=name, kind="norm", tokens=tokens, first=first, heads=heads, kv_heads=kv_heads, dim=dim, dims=dims,
                interleaved=interleaved, dtype=dtype)


def _append(name, seqs, prefix, shortest, longest, heads, kv_heads, dim, dims, interleaved, norm, dtype, page):
    return dict(name=name, kind="append", seqs=seqs, prefix=prefix, shortest=shortest, longest=longest, heads=heads,
                kv_heads=kv_heads, dim=dim, dims=dims, interleaved=interleaved, norm=norm, dtype=dtype, page=page)


def _prompt(name, seqs, shortest, longest, prefix, heads, kv_heads, dim, dtype, causal, cap, bias):
    return dict(name=name, kind="prompt", seqs=seqs, shortest=shortest, longest=longest, prefix=prefix, heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal, cap=cap, bias=bias)


def _step(name, seqs, prefix, shortest, longest, new, heads, kv_heads, dim, dtype, page, cap, bias):
    return dict(name=name, kind="step", seqs=seqs, prefix=prefix, shortest=shortest, longest=longest, new=new,
                heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, cap=cap, bias=bias)


def listed():
    return [
        # The next token of one conversation through a small model: launches and latency count.
        _rotate("rotate_token", 1, 776, 16, 64, 64, False, "", "fp16"),
        # The far end of a long context: part of each head, neighbours in pairs, frequencies scaled.
        _rotate("rotate_far", 20_011, 100_000, 20, 80, 32, True, "turns", "bf16"),
        # The next tokens of a batch.
        _norm("norm_step", 48, 6000, 32, 8, 128, 128, False, "bf16"),
        # Prompts of odd length, a head size that is no power of two, half of each head rotated.
        _norm("norm_odd", 3001, 0, 20, 4, 80, 40, False, "fp16"),
        # Passages set one behind another into one long prompt.
        _norm("norm_prompt", 12_000, 0, 32, 8, 128, 128, False, "bf16"),
        # The next token of a single short conversation: latency.
        _append("append_token", 1, 776, 1, 1, 16, 4, 64, 64, False, False, "fp16", 32),
        # The next tokens of many questions over the same passages.
        _append("append_step", 64, 8000, 1, 1, 32, 8, 128, 128, False, True, "bf16", 64),
        # Prompts of very different lengths into the cache, one token and none among them; pairs of neighbours.
        _append("append_prompts", 24, 0, 0, 2000, 20, 4, 80, 80, True, True, "bf16", 64),
        # A batch of passages through an embedding model that knows positions by distance alone.
        _prompt("prompt_distance", 64, 40, 512, 0, 12, 12, 64, "fp16", False, 0.0, True),
        # Passages that are seen in both directions and a question behind them, scores capped.
        _prompt("prompt_prefix", 1, 8000, 8000, 6000, 32, 8, 128, "bf16", True, 50.0, False),
        # The next token of a single short conversation, biased by distance: latency.
        _step("step_distance", 1, 0, 777, 777, 1, 16, 4, 64, "fp16", 32, 0.0, True),
        # The next tokens of a batch with nothing in common, scores capped.
        _step("step_capped", 48, 0, 100, 6000, 1, 32, 8, 128, "bf16", 64, 30.0, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn_dims(rng, dim):
    """Rotated channels: mostly all, or a half, a quarter, or another even number of them."""
    return rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])


def draw(rng):
    kind = rng.choice(["rotate", "norm", "append", "append", "prompt", "prompt", "step", "step"])
    dim = rng.choice([64, 80, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([32, 64, 128])
    dims, interleaved = _drawn_dims(rng, dim), rng.random() < 0.4
    cap, bias = rng.choice([(30.0, False), (50.0, False), (0.0, True), (0.0, True), (50.0, True)])
    if kind in ("rotate", "norm"):
        while True:
            tokens, first = _log_int(rng, 1, 20_011), rng.choice([0, _log_int(rng, 1, 1_000_000)])
            if tokens * (heads + kv_heads) * dim <= 12_000 * 40 * 128:
                break
        if kind == "rotate":
            scaling = rng.choice(["", "linear", "base", "turns"])
            c = _rotate("", tokens, first, heads, dim, max(dims, 4), interleaved, scaling, dtype)
        else:
            c = _norm("", tokens, first, heads, kv_heads, dim, dims, interleaved, dtype)
    elif kind == "append":
        while True:
            seqs, prefix = _log_int(rng, 1, 64), rng.choice([0, 1, 1]) * _log_int(rng, 1, 100_000)
            longest = rng.choice([1, _log_int(rng, 2, 2000)])
            if seqs * longest * (heads + 8 * kv_heads) * dim <= 24 * 1000 * 52 * 80:
                break
        c = _append("", seqs, prefix, rng.choice([0, 1, longest]), longest, heads, kv_heads, dim, dims, interleaved,
                    rng.random() < 0.5, dtype, page)
    elif kind == "prompt":
        while True:
            seqs, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 8000)
            if seqs * heads * longest ** 2 <= 32 * 8000 ** 2:
                break
        causal = rng.random() < 0.6
        prefix = rng.choice([0, _log_int(rng, 1, longest)]) if causal else 0
        c = _prompt("", seqs, rng.choice([0, 1, max(1, longest // 8), longest]), longest, prefix, heads, kv_heads, dim,
                    dtype, causal, cap, bias)
    else:
        while True:
            seqs, prefix = _log_int(rng, 1, 64), rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, 100_000)
            longest = _log_int(rng, 5, 6000)
            new = rng.choice([1, 1, 1, min(longest, _log_int(rng, 2, 60))])
            if seqs * heads * new * (prefix + longest) <= 64 * 32 * 100_000 and seqs * longest <= 48 * 6000:
                break
        c = _step("", seqs, prefix, rng.choice([new, max(new, longest // 8), longest]), longest, new, heads, kv_heads,
                  dim, dtype, page, cap, bias)
    del c["name"]
    return c


def _lengths(case):
    """The lengths of a case's sequences: the case's alone, so that its work is known; the longest is among them."""
    r = random.Random("%(kind)s %(seqs)d %(shortest)d %(longest)d %(dim)d" % case)
    lengths = [r.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lengths[r.randrange(case["seqs"])] = case["longest"]
    return lengths


# ---- inputs ----------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed((seed * 1_000_003 + 29) & 0x7FFFFFFF)


def _heads(g, rows, heads, dim, dtype, offset=0.0):
    """Rows of a projection: normal values, for keys with an offset of each channel, as trained keys have."""
    x = torch.randn(rows, heads, dim, generator=g, device="cuda")
    if offset:
        x += offset * torch.randn(heads, dim, generator=g, device="cuda")
    return x.to(dtype)


def _weight(g, dim, dtype):
    """A norm's weight: near one, as trained ones are."""
    return (1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# How a case's frequencies are made: base, and what a context of 131,072 tokens does to a model of 8,192.
BASE, FACTOR, ORIGINAL, LOW, HIGH = 500_000.0, 16.0, 8192, 1.0, 32.0
MAGNITUDE = 0.1 * math.log(FACTOR) + 1.0  # of the scaling by turns


def _rotary(case):
    scaling = case.get("scaling", "")
    if scaling == "turns":
        return _context().rotary(case["dims"], base=BASE, interleaved=case["interleaved"], scaling="turns",
                                 factor=FACTOR, original_length=ORIGINAL, low=LOW, high=HIGH, magnitude=MAGNITUDE)
    if scaling:
        return _context().rotary(case["dims"], base=BASE, interleaved=case["interleaved"], scaling=scaling,
                                 factor=FACTOR)
    return _context().rotary(case["dims"], base=BASE, interleaved=case["interleaved"])


def _frequencies(case):
    """Radians a position of each pair of channels, in 64 bits, and the factor of what is rotated."""
    dims, scaling = case["dims"], case.get("scaling", "")
    base = BASE * FACTOR ** (dims / (dims - 2)) if scaling == "base" else BASE
    f = base ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    if scaling == "linear":
        f = f / FACTOR
    if scaling == "turns":
        share = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0.0, 1.0)
        return f * (share + (1 - share) / FACTOR), MAGNITUDE
    return f, 1.0


def prepare(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    return {"rotate": _prepare_rotate, "norm": _prepare_norm, "append": _prepare_append, "prompt": _prepare_prompt,
            "step": _prepare_step}[case["kind"]](case, g, dtype)


def _prepare_rotate(case, g, dtype):
    x = _heads(g, case["tokens"], case["heads"], case["dim"], dtype)
    s = {"case": case, "x": x, "out": torch.zeros_like(x),
         "positions": torch.arange(case["first"], case["first"] + case["tokens"], device="cuda")}
    if own:
        s["ctx"], s["rotary"] = _context(), _rotary(case)
    else:
        s["frequencies"], s["magnitude"] = _frequencies(case)
    return s


def _prepare_norm(case, g, dtype):
    tokens, h, kv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    qkv = torch.cat([_heads(g, tokens, h, dim, dtype), _heads(g, tokens, kv, dim, dtype, 1.0),
                     _heads(g, tokens, kv, dim, dtype)], dim=1)
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "q_weight": _weight(g, dim, dtype),
         "k_weight": _weight(g, dim, dtype), "q_out": torch.zeros(tokens, h, dim, dtype=dtype, device="cuda"),
         "k_out": torch.zeros(tokens, kv, dim, dtype=dtype, device="cuda"),
         "positions": torch.arange(case["first"], case["first"] + tokens, device="cuda")}
    if own:
        s["ctx"], s["rotary"] = _context(), _rotary(case)
    else:
        s["frequencies"], s["magnitude"] = _frequencies(case)
    return s


def _prepare_append(case, g, dtype):
    n, prefix, page, dim, lengths = case["seqs"], case["prefix"], case["page"], case["dim"], _lengths(case)
    h, kv, tokens = case["heads"], case["kv_heads"], sum(lengths)
    qkv = torch.cat([_heads(g, tokens, h, dim, dtype), _heads(g, tokens, kv, dim, dtype, 1.0),
                     _heads(g, tokens, kv, dim, dtype)], dim=1)
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:],
         "q_weight": _weight(g, dim, dtype) if case["norm"] else None,
         "k_weight": _weight(g, dim, dtype) if case["norm"] else None,
         "q_out": torch.zeros(tokens, h, dim, dtype=dtype, device="cuda"),
         "k_out": torch.zeros(tokens, kv, dim, dtype=dtype, device="cuda"),
         "v_out": torch.zeros(tokens, kv, dim, dtype=dtype, device="cuda")}
    pages = -(-prefix // page) + sum(-(-m // page) + 2 for m in lengths)
    if own:
        cache = _context().kv_cache(1, pages, page, kv, dim, case["dtype"])
        root = cache.sequence()
        cache.extend([root], [prefix])
        seqs = cache.fork(root, n)
        cache.extend(seqs, lengths)
        s["cache"], s["plan"], s["rotary"] = cache, cache.plan(seqs, lengths), _rotary(case)
    else:
        # The pages themselves, and where in them the new tokens go: the prefix's last page is copied for each sequence.
        s["frequencies"], s["magnitude"] = _frequencies(case)
        s["pool"] = torch.zeros(2, pages * page, kv, dim, dtype=dtype, device="cuda")
        whole, tail, at, slots, positions = prefix // page, prefix % page, -(-prefix // page), [], []
        for m in lengths:
            slots += range(at * page + tail, at * page + tail + m)
            positions += range(prefix, prefix + m)
            at += -(-(tail + m) // page)
        s["slots"], s["positions"] = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in (slots, positions))
    return s


def _slopes(heads):
    """One for each head, from steep to nearly flat."""
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads)


def _prepare_prompt(case, g, dtype):
    h, kv, dim, lengths = case["heads"], case["kv_heads"], case["dim"], _lengths(case)
    tokens = sum(lengths)
    qkv = torch.cat([_heads(g, tokens, h, dim, dtype), _heads(g, tokens, kv, dim, dtype, 1.0),
                     _heads(g, tokens, kv, dim, dtype)], dim=1)
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:],
         "out": torch.zeros(tokens, h, dim, dtype=dtype, device="cuda"), "lengths": _int32(lengths),
         "longest": max(lengths), "slopes": _slopes(h) if case["bias"] else None}
    if own:
        prefixes = [min(case["prefix"], m) for m in lengths] if case["prefix"] else None
        s["ctx"] = _context()
        s["plan"] = s["ctx"].prompt_plan(lengths, h, kv, causal=case["causal"], prefixes=prefixes)
    return s


def _prepare_step(case, g, dtype):
    h, kv, dim, new, lengths = case["heads"], case["kv_heads"], case["dim"], case["new"], _lengths(case)
    n, prefix, tokens = case["seqs"], case["prefix"], sum(lengths)
    q = _heads(g, n * new, h, dim, dtype)
    k, v = _heads(g, prefix + tokens, kv, dim, dtype, 1.0), _heads(g, prefix + tokens, kv, dim, dtype)
    s = {"case": case, "q": q, "k_prefix": k[:prefix], "v_prefix": v[:prefix], "k_own": k[prefix:], "v_own": v[prefix:],
         "out": torch.zeros(n * new, h, dim, dtype=dtype, device="cuda"), "lengths": _int32(lengths),
         "longest": max(lengths), "slopes": _slopes(h) if case["bias"] else None}
    if own:
        page = case["page"]
        pages = -(-prefix // page) + sum(-(-m // page) + 2 for m in lengths)
        cache = _context().kv_cache(1, pages, page, kv, dim, case["dtype"])
        root = cache.sequence()
        cache.extend([root], [prefix])
        plan = cache.plan([root], [prefix])
        cache.write_async(plan, s["k_prefix"], s["v_prefix"])
        seqs = cache.fork(root, n)
        cache.extend(seqs, lengths)
        plan = cache.plan(seqs, lengths)
        cache.write_async(plan, s["k_own"], s["v_own"])
        s["cache"], s["plan"] = cache, cache.plan(seqs, [new] * n, heads=h)
    return s


# ---- one pass --------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "norm": _own_norm, "append": _own_append, "prompt": _own_prompt,
                "step": _own_step}[kind](state)
    return {"rotate": _plain_rotate, "norm": _plain_norm, "append": _plain_append, "prompt": _plain_prompt,
            "step": _plain_step}[kind](state)


def _own_rotate(s):
    s["ctx"].rotate_async(s["rotary"], s["positions"], s["x"], s["out"])
    return s["out"]


def _own_norm(s):
    s["ctx"].norm_rotate_async(s["rotary"], s["positions"], s["q"], s["q_out"], s["k"], s["k_out"], s["q_weight"],
                               s["k_weight"], eps=EPS)
    return s["q_out"], s["k_out"]


def _own_append(s):
    s["cache"].append_async(s["plan"], s["k"], s["v"], rotary=s["rotary"], k_weight=s["k_weight"], q=s["q"],
                            q_out=s["q_out"], q_weight=s["q_weight"], eps=EPS)
    s["cache"].read_async(s["plan"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_prompt(s):
    s["ctx"].prompt_attention_async(s["plan"], s["q"], s["k"], s["v"], s["out"], cap=s["case"]["cap"],
                                    slopes=s["slopes"])
    return s["out"]


def _own_step(s):
    s["cache"].attention_async(s["plan"], s["q"], s["out"], cap=s["case"]["cap"], slopes=s["slopes"])
    return s["out"]


def _rotated(s, x):
    """x (tokens, heads, dim) in 32 bits, its first channels turned by position."""
    dims, half = s["case"]["dims"], s["case"]["dims"] // 2
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (s["magnitude"] * f(angle)[:, None].float() for f in (torch.cos, torch.sin))
    if s["case"]["interleaved"]:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:dims]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., dims:]], dim=-1)


def _normed(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * x.square().mean(-1, keepdim=True).add(EPS).rsqrt() * weight.float()


def _plain_rotate(s):
    s["out"].copy_(_rotated(s, s["x"].float()))
    return s["out"]


def _plain_norm(s):
    s["q_out"].copy_(_rotated(s, _normed(s["q"], s["q_weight"])))
    s["k_out"].copy_(_rotated(s, _normed(s["k"], s["k_weight"])))
    return s["q_out"], s["k_out"]


def _plain_append(s):
    pool, slots = s["pool"], s["slots"]
    s["q_out"].copy_(_rotated(s, _normed(s["q"], s["q_weight"])))
    pool[0][slots] = _rotated(s, _normed(s["k"], s["k_weight"])).to(pool.dtype)
    pool[1][slots] = s["v"]
    s["k_out"].copy_(pool[0][slots])
    s["v_out"].copy_(pool[1][slots])
    return s["q_out"], s["k_out"], s["v_out"]


def _softmax_values(x, v):
    """Softmax of the last axis of x, -inf where masked, times v; rows with nothing to see give zeros."""
    top = x.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v).div_(total.masked_fill_(total == 0, 1.0))


def _capped(x, cap):
    """In place: scores within -cap to cap."""
    return x.div_(cap).tanh_().mul_(cap) if cap else x


def _rows_of(lengths, longest):
    """For sequences packed one behind another: (n, longest) row numbers, and which of them are there."""
    place = torch.arange(longest, device="cuda")
    there = place < lengths[:, None]
    start = torch.cumsum(lengths, 0) - lengths
    return (start[:, None] + place).masked_fill_(~there, 0), there


def _plain_prompt(s):
    case, dim, kv = s["case"], s["case"]["dim"], s["case"]["kv_heads"]
    lengths = s["lengths"].long()
    rows, there = _rows_of(lengths, s["longest"])
    n, m = rows.shape
    group = case["heads"] // kv
    q = s["q"].float()[rows].view(n, m, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * m, dim)
    k = s["k"].float()[rows].permute(0, 2, 3, 1).contiguous()
    v = s["v"].float()[rows].permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(n, kv, group, m, m)
    x = _capped(x, case["cap"])
    place = torch.arange(m, device="cuda")
    if case["bias"]:
        distance = (place[None, :] - place[:, None]).abs().float()
        for j in range(case["heads"]):
            x[:, j // group, j % group].addcmul_(distance, s["slopes"][j], value=-1.0)
    x.masked_fill_(~there[:, None, None, None, :], -math.inf)
    if case["causal"]:
        x.masked_fill_((place[None, :] > place[:, None]) & (place >= case["prefix"])[None, :], -math.inf)
    y = _softmax_values(x.view(n, kv, group * m, m), v)
    y = y.view(n, kv, group, m, dim).permute(0, 3, 1, 2, 4).reshape(n, m, kv * group, dim)
    s["out"].copy_(y[there])
    return s["out"]


def _plain_step(s):
    case, dim, kv, new = s["case"], s["case"]["dim"], s["case"]["kv_heads"], s["case"]["new"]
    lengths, prefix, n = s["lengths"].long(), case["prefix"], case["seqs"]
    rows, there = _rows_of(lengths, s["longest"])
    m, group = rows.shape[1], case["heads"] // kv
    q = s["q"].float().view(n, new, kv, group, dim).permute(2, 0, 3, 1, 4).mul(1.0 / math.sqrt(dim))
    # The shared keys once for all rows, each sequence's own keys for its rows.
    far = torch.matmul(q.reshape(kv, n * group * new, dim), s["k_prefix"].float().permute(1, 2, 0).contiguous())
    near = torch.matmul(q.reshape(kv, n, group * new, dim), s["k_own"].float()[rows].permute(2, 0, 3, 1).contiguous())
    x = torch.cat([far.view(kv, n, group, new, prefix), near.view(kv, n, group, new, m)], dim=-1)
    x = _capped(x, case["cap"])
    last = prefix + lengths[:, None] - new + torch.arange(new, device="cuda")  # the newest key that each row sees
    back = last[:, :, None] - torch.arange(prefix + m, device="cuda")
    if case["bias"]:
        x.sub_(back[None, :, None].float() * s["slopes"].view(kv, 1, group, 1, 1))
    x.masked_fill_((back < 0)[None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x[..., :prefix].reshape(kv, n * group * new, prefix),
                     s["v_prefix"].float().transpose(0, 1).contiguous())
    y = y.view(kv, n, group * new, dim)
    own_v = s["v_own"].float()[rows].permute(2, 0, 1, 3).contiguous()
    y = y + torch.matmul(x[..., prefix:].reshape(kv, n, group * new, m), own_v)
    y = y.view(kv, n, group, new, dim).div_(total).permute(1, 3, 0, 2, 4)
    s["out"].copy_(y.reshape(n * new, kv * group, dim))
    return s["out"]


# ---- what a pass needs, and how exact it is ---------------------------------


def work(case):
    kind, h, dim = case["kind"], case["heads"], case["dim"]
    if kind == "rotate":
        return {"bytes": case["tokens"] * (2 * 2 * h * dim + 8), "flops": 3.0 * case["tokens"] * h * case["dims"]}
    kv = case["kv_heads"]
    if kind == "norm":
        return {"bytes": case["tokens"] * (2 * 2 * (h + kv) * dim + 8),
                "flops": case["tokens"] * (h + kv) * (4.0 * dim + 3.0 * case["dims"])}
    lengths = _lengths(case)
    if kind == "append":
        # q, k, v read; q and the pages written; the pages read again and written out.
        each = 3.0 * case["dims"] + (4.0 * dim if case["norm"] else 0.0)
        return {"bytes": 2 * sum(lengths) * (2 * h + 4 * 2 * kv) * dim, "flops": sum(lengths) * (h + kv) * each}
    if kind == "prompt":
        if case["causal"]:
            prefixes = [min(case["prefix"], m) for m in lengths]
            pairs = sum(m * (m + 1) // 2 + p * (p - 1) // 2 for m, p in zip(lengths, prefixes))
        else:
            pairs = sum(m * m for m in lengths)
        return {"bytes": 2 * sum(lengths) * (2 * h + 2 * kv) * dim, "flops": 4.0 * h * dim * pairs}
    new = case["new"]
    pairs = sum(new * (case["prefix"] + m) - new * (new - 1) // 2 for m in lengths)
    return {"bytes": 2 * (case["prefix"] + sum(lengths)) * 2 * kv * dim + 2 * 2 * case["seqs"] * new * h * dim,
            "flops": 4.0 * h * dim * pairs}


def _exact_rotation(case, x, positions):
    """x in 64 bits as complex numbers times the unit ones of their angles."""
    dims, scaling = case["dims"], case.get("scaling", "")
    pairs = torch.arange(dims // 2, dtype=torch.float64, device="cuda")
    base = math.log(BASE)
    if scaling == "base":
        base += dims / (dims - 2) * math.log(FACTOR)
    f, magnitude = torch.exp(-2.0 * pairs / dims * base), 1.0
    if scaling == "linear":
        f /= FACTOR
    elif scaling == "turns":
        w = torch.clip((f * ORIGINAL / math.tau - LOW) / (HIGH - LOW), 0, 1)
        f, magnitude = f * w + f / FACTOR * (1 - w), MAGNITUDE
    turn = torch.polar(torch.full((len(positions), dims // 2), magnitude, dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), f))
    y = x.clone()
    first, second = ((slice(0, dims, 2), slice(1, dims, 2)) if case["interleaved"]
                     else (slice(0, dims // 2), slice(dims // 2, dims)))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_norm(x, weight):
    if weight is None:
        return x.double()
    x = x.double()
    return x * weight.double() / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    """The outputs in 64 bits, from the definition: attention sequence by sequence and head by head."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotate":
        return _exact_rotation(case, s["x"].double(), s["positions"])
    if kind == "norm":
        return tuple(_exact_rotation(case, _exact_norm(s[x], s[x + "_weight"]), s["positions"]) for x in "qk")
    lengths, h, kv, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        at = torch.cat([case["prefix"] + torch.arange(m, device="cuda") for m in lengths])
        q, k = (_exact_rotation(case, _exact_norm(s[x], s[x + "_weight"]), at) for x in "qk")
        return q, k, s["v"].double()
    group = h // kv
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, m in enumerate(lengths):
        if kind == "prompt":
            q, k, v = (s[x][at:at + m].double() for x in "qkv")
            first, rows, o = 0, m, out[at:at + m]
        else:
            new = case["new"]
            q = s["q"][b * new:(b + 1) * new].double()
            k = torch.cat([s["k_prefix"], s["k_own"][at:at + m]]).double()
            v = torch.cat([s["v_prefix"], s["v_own"][at:at + m]]).double()
            first, rows, o = case["prefix"] + m - new, new, out[b * new:(b + 1) * new]
        at += m
        if not rows:
            continue
        ahead = torch.arange(k.shape[0], device="cuda")[None, :] - torch.arange(first, first + rows, device="cuda")[:, None]
        hide = None
        if kind == "step" or case["causal"]:
            hide = ahead > 0
            if kind == "prompt":
                hide[:, :case["prefix"]] = False
        for j in range(h):
            w = (q[:, j] @ k[:, j // group].T) / math.sqrt(dim)
            if case["cap"]:
                w = case["cap"] * torch.tanh(w / case["cap"])
            if case["bias"]:
                w -= s["slopes"][j].double() * ahead.abs()
            if hide is not None:
                w.masked_fill_(hide, -math.inf)
            o[:, j] = torch.softmax(w, dim=1) @ v[:, j // group]
    return out
