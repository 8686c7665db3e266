"""Timed calls of the attention and cache operators: what is run, on which inputs, their plain forms and exact values.

Three kinds of call, as a program that answers questions over the passages a search found makes them:

- ``prompt``: attention over packed sequences of different lengths (passages or questions through a model's layer),
  causal or not, with grouped heads; q, k and v are views of one fused projection;
- ``step``: attention of each sequence's newest tokens over a paged cache, where the sequences of a batch share a long
  prefix (the passages) or nothing;
- ``fork`` and ``compact``: pages of the cache. ``fork`` makes the sequences of several questions from one that holds
  the passages, appends to each, reads back what each holds beyond the shared pages, and frees them. ``compact`` brings
  sequences in behind one that then ends, closes the gap, and takes the sequences out again.

Where ``own`` is false the operators run in their plain form: elementary torch operations in 32 bits.
"""
from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


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


def _prompt(name, seqs, shortest, longest, heads, kv_heads, dim, dtype, causal=True):
    return dict(name=name, kind="prompt", seqs=seqs, shortest=shortest, longest=longest, heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal)


def _step(name, seqs, prefix, shortest, longest, new, heads, kv_heads, dim, dtype, page):
    return dict(name=name, kind="step", seqs=seqs, prefix=prefix, shortest=shortest, longest=longest, new=new,
                heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page)


def _pages(name, kind, layers, seqs, tokens, new, kv_heads, dim, dtype, page):
    return dict(name=name, kind=kind, layers=layers, seqs=seqs, tokens=tokens, new=new, kv_heads=kv_heads, dim=dim,
                dtype=dtype, page=page)


def listed():
    return [
        # One question through a layer of a small model: launches and latency count.
        _prompt("prompt_question", 1, 23, 23, 16, 4, 64, "fp16"),
        # A batch of passages through an embedding model, each token seeing its whole passage.
        _prompt("prompt_passages", 64, 40, 512, 12, 12, 64, "fp16", causal=False),
        # Prompts of very different lengths in one batch, one token and none among them; a head size that is no
        # power of two.
        _prompt("prompt_ragged", 24, 0, 2000, 20, 4, 80, "bf16"),
        # Passages set one behind another into one long prompt: matrix-core bound.
        _prompt("prompt_long", 1, 12_000, 12_000, 32, 8, 128, "bf16"),
        # The next token of a single short conversation: latency.
        _step("step_one", 1, 0, 777, 777, 1, 16, 4, 64, "fp16", 32),
        # The next tokens of a batch with nothing in common, of different lengths: HBM bound.
        _step("step_private", 48, 0, 100, 6000, 1, 32, 8, 128, "bf16", 64),
        # The next tokens of many questions over the same passages.
        _step("step_shared", 64, 8000, 1, 300, 1, 32, 8, 128, "fp16", 64),
        # A few questions over a whole collection of passages: a long axis to split.
        _step("step_collection", 8, 100_003, 1, 500, 1, 32, 8, 128, "bf16", 128),
        # The questions themselves, several tokens each, over the passages' cache.
        _step("step_questions", 32, 4001, 5, 60, 5, 20, 4, 80, "bf16", 64),
        # Two answers to one question: a page each.
        _pages("fork_small", "fork", 4, 2, 77, 1, 4, 64, "fp16", 32),
        # Many questions over the same passages.
        _pages("fork_questions", "fork", 16, 64, 8000, 9, 8, 128, "bf16", 64),
        # Sequences brought into the cache, the gap below them closed, and taken out again.
        _pages("compact", "compact", 16, 12, 1500, 700, 8, 128, "bf16", 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "step", "step", "fork", "compact"])
    dim = rng.choice([64, 80, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([32, 64, 128])
    if kind == "prompt":
        while True:
            seqs, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 12_000)
            if seqs * heads * longest ** 2 <= 32 * 12_000 ** 2:
                break
        c = _prompt("", seqs, rng.choice([0, 1, max(1, longest // 8), longest]), longest, heads, kv_heads, dim, dtype,
                    rng.random() < 0.7)
    elif kind == "step":
        while True:
            seqs, prefix = _log_int(rng, 1, 64), rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, 100_000)
            longest = _log_int(rng, 5, 6000)
            new = rng.choice([1, 1, 1, min(longest, _log_int(rng, 2, 60))])
            if seqs * heads * new * (prefix + longest) <= 64 * 32 * 100_000 and seqs * longest <= 48 * 6000:
                break
        c = _step("", seqs, prefix, rng.choice([new, max(new, longest // 8), longest]), longest, new, heads, kv_heads,
                  dim, dtype, page)
    else:
        while True:
            layers, seqs = _log_int(rng, 1, 16), _log_int(rng, 1, 64)
            tokens, new = _log_int(rng, 1, 8000), _log_int(rng, 1, 700)
            if layers * (tokens + seqs * (new + page)) * kv_heads * dim <= 16 * 20_000 * 8 * 128:
                break
        c = _pages("", kind, layers, seqs, tokens, new, kv_heads, dim, dtype, page)
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
    return torch.Generator(device="cuda").manual_seed((seed * 1_000_003 + 17) & 0x7FFFFFFF)


def _heads(g, rows, heads, dim, dtype, offset=0.0):
    """Rows of a projection: normal values, for keys with an offset of each channel, as trained keys have."""
    x = torch.randn(rows, heads, dim, generator=g, device="cuda")
    if offset:
        x += offset * torch.randn(heads, dim, generator=g, device="cuda")
    return x.to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    return {"prompt": _prepare_prompt, "step": _prepare_step, "fork": _prepare_pages,
            "compact": _prepare_pages}[case["kind"]](case, g, dtype)


def _prepare_prompt(case, g, dtype):
    h, kv, dim, lengths = case["heads"], case["kv_heads"], case["dim"], _lengths(case)
    tokens = sum(lengths)
    qkv = torch.cat([_heads(g, tokens, h, dim, dtype), _heads(g, tokens, kv, dim, dtype, 1.0),
                     _heads(g, tokens, kv, dim, dtype)], dim=1)
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:],
         "out": torch.zeros(tokens, h, dim, dtype=dtype, device="cuda"), "lengths": _int32(lengths),
         "longest": max(lengths)}
    if own:
        s["ctx"] = _context()
        s["plan"] = s["ctx"].prompt_plan(lengths, h, kv, causal=case["causal"])
    return s


def _prepare_step(case, g, dtype):
    h, kv, dim, new, lengths = case["heads"], case["kv_heads"], case["dim"], case["new"], _lengths(case)
    n, prefix, tokens = case["seqs"], case["prefix"], sum(lengths)
    q = _heads(g, n * new, h, dim, dtype)
    k, v = _heads(g, prefix + tokens, kv, dim, dtype, 1.0), _heads(g, prefix + tokens, kv, dim, dtype)
    s = {"case": case, "q": q, "k_prefix": k[:prefix], "v_prefix": v[:prefix], "k_own": k[prefix:], "v_own": v[prefix:],
         "out": torch.zeros(n * new, h, dim, dtype=dtype, device="cuda"), "lengths": _int32(lengths),
         "longest": max(lengths)}
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


def _prepare_pages(case, g, dtype):
    layers, n, tokens, new = case["layers"], case["seqs"], case["tokens"], case["new"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    old = 2 * layers * tokens
    filled = _heads(g, old, kv, dim, dtype).view(2, layers, tokens, kv, dim)
    fresh = _heads(g, 2 * layers * n * new, kv, dim, dtype).view(2, layers, n * new, kv, dim)
    tail = tokens % page if case["kind"] == "fork" else 0
    pages = -(-tokens // page) + n * -(-(tail + new) // page)
    if case["kind"] == "compact":
        pages += -(-tokens // page)
    s = {"case": case, "filled": filled, "fresh": fresh, "pages": pages,
         "out": torch.zeros(2, layers, n * (tail + new), kv, dim, dtype=dtype, device="cuda")}
    if own:
        cache = _context().kv_cache(layers, pages, page, kv, dim, case["dtype"])
        root = cache.sequence()
        cache.extend([root], [tokens])
        cache.write_async(cache.plan([root], [tokens]), filled[0], filled[1])
        s["cache"], s["root"] = cache, root
    else:
        # The pages themselves, the sequence's in pages 0 and on.
        pool = torch.zeros(2, layers, pages, page, kv, dim, dtype=dtype, device="cuda")
        pool.view(2, layers, pages * page, kv, dim)[:, :, :tokens] = filled
        s["pool"] = pool
    return s


# ---- one pass --------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"prompt": _own_prompt, "step": _own_step, "fork": _own_fork, "compact": _own_compact}[kind](state)
    return {"prompt": _plain_prompt, "step": _plain_step, "fork": _plain_fork, "compact": _plain_compact}[kind](state)


def _own_prompt(s):
    s["ctx"].prompt_attention_async(s["plan"], s["q"], s["k"], s["v"], s["out"])
    return s["out"]


def _own_step(s):
    s["cache"].attention_async(s["plan"], s["q"], s["out"])
    return s["out"]


def _own_fork(s):
    cache, case, out = s["cache"], s["case"], s["out"]
    n, new = case["seqs"], case["new"]
    tail = case["tokens"] % case["page"]
    seqs = cache.fork(s["root"], n)
    cache.extend(seqs, [new] * n)
    cache.write_async(cache.plan(seqs, [new] * n), s["fresh"][0], s["fresh"][1])
    cache.read_async(cache.plan(seqs, [tail + new] * n), out[0], out[1])
    tables = cache.pages(seqs).astype(np.int32)
    cache.free(seqs)
    return out, tables


def _own_compact(s):
    cache, case, out = s["cache"], s["case"], s["out"]
    n, new = case["seqs"], case["new"]
    gap = cache.sequence()
    cache.extend([gap], [case["tokens"]])
    seqs = cache.sequences(n)
    cache.extend(seqs, [new] * n)
    cache.write_async(cache.plan(seqs, [new] * n), s["fresh"][0], s["fresh"][1])
    cache.free([gap])
    cache.compact()
    cache.read_async(cache.plan(seqs, [new] * n), out[0], out[1])
    tables = cache.pages(seqs).astype(np.int32)
    cache.free(seqs)
    return out, tables


def _softmax_values(x, v):
    """Softmax of the last axis of x, -inf where masked, times v; rows with nothing to see give zeros."""
    top = x.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v).div_(total.masked_fill_(total == 0, 1.0))


def _rows_of(lengths, longest):
    """For sequences packed one behind another: (n, longest) row numbers, and which of them are there."""
    place = torch.arange(longest, device="cuda")
    there = place < lengths[:, None]
    start = torch.cumsum(lengths, 0) - lengths
    return (start[:, None] + place).masked_fill_(~there, 0), there


def _plain_prompt(s):
    case, dim, kv = s["case"], s["case"]["dim"], s["case"]["kv_heads"]
    rows, there = _rows_of(s["lengths"].long(), s["longest"])
    n, m = rows.shape
    group = case["heads"] // kv
    q = s["q"].float()[rows].view(n, m, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * m, dim)
    k = s["k"].float()[rows].permute(0, 2, 3, 1)
    v = s["v"].float()[rows].permute(0, 2, 1, 3)
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(n, kv, group, m, m)
    x.masked_fill_(~there[:, None, None, None, :], -math.inf)
    if case["causal"]:
        place = torch.arange(m, device="cuda")
        x.masked_fill_(place[None, :] > place[:, None], -math.inf)
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
    far = torch.matmul(q.reshape(kv, n * group * new, dim), s["k_prefix"].float().permute(1, 2, 0))
    near = torch.matmul(q.reshape(kv, n, group * new, dim), s["k_own"].float()[rows].permute(2, 0, 3, 1))
    near = near.view(kv, n, group, new, m)
    last = lengths[:, None] - new + torch.arange(new, device="cuda")  # the newest key that each row sees
    hidden = torch.arange(m, device="cuda") > last[:, :, None]
    near.masked_fill_(hidden[None, :, None], -math.inf)
    x = torch.cat([far.view(kv, n, group, new, prefix), near], dim=-1)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x[..., :prefix].reshape(kv, n * group * new, prefix), s["v_prefix"].float().transpose(0, 1))
    y = y.view(kv, n, group * new, dim)
    y = y + torch.matmul(x[..., prefix:].reshape(kv, n, group * new, m), s["v_own"].float()[rows].permute(2, 0, 1, 3))
    y = y.view(kv, n, group, new, dim).div_(total).permute(1, 3, 0, 2, 4)
    s["out"].copy_(y.reshape(n * new, kv * group, dim))
    return s["out"]


def _plain_fork(s):
    case, pool, page = s["case"], s["pool"], s["case"]["page"]
    n, tokens, new = case["seqs"], case["tokens"], case["new"]
    whole, tail = tokens // page, tokens % page
    more = -(-(tail + new) // page)  # pages of its own that each sequence needs
    base = -(-tokens // page)
    ids = base + np.arange(n * more, dtype=np.int32).reshape(n, more)
    place = torch.as_tensor(ids, device="cuda").long()
    if tail:
        pool[:, :, place[:, 0]] = pool[:, :, whole:whole + 1]
    flat = pool.view(*pool.shape[:2], -1, *pool.shape[4:])
    at = torch.arange(tail + new, device="cuda")
    slots = place[:, at // page] * page + at % page
    flat[:, :, slots[:, tail:].reshape(-1)] = s["fresh"]
    s["out"].copy_(flat[:, :, slots.reshape(-1)])
    shared = np.tile(np.arange(whole, dtype=np.int32), (n, 1))
    return s["out"], np.concatenate([shared, ids], axis=1).reshape(-1)


def _plain_compact(s):
    case, pool, page = s["case"], s["pool"], s["case"]["page"]
    n, tokens, new = case["seqs"], case["tokens"], case["new"]
    base, each = -(-tokens // page), -(-new // page)
    gap = base  # pages base .. base + gap - 1 end before the sequences' own do
    ids = base + gap + np.arange(n * each, dtype=np.int32)
    flat = pool.view(*pool.shape[:2], -1, *pool.shape[4:])
    at = torch.arange(new, device="cuda")
    place = torch.as_tensor(ids, device="cuda").long().view(n, each)
    flat[:, :, (place[:, at // page] * page + at % page).reshape(-1)] = s["fresh"]
    # The pages past the number of live ones go, lowest first, to the free ones below it.
    live = base + n * each
    moved = ids >= live
    holes = base + np.arange(moved.sum(), dtype=np.int32)
    pool[:, :, torch.as_tensor(holes, device="cuda").long()] = pool[:, :, place.view(-1)[int(n * each - moved.sum()):]]
    ids[moved] = holes
    place = torch.as_tensor(ids, device="cuda").long().view(n, each)
    s["out"].copy_(flat[:, :, (place[:, at // page] * page + at % page).reshape(-1)])
    return s["out"], ids


# ---- what a pass needs, and how exact it is ---------------------------------


def work(case):
    kind, kv, dim = case["kind"], case["kv_heads"], case["dim"]
    if kind == "prompt":
        lengths, h = _lengths(case), case["heads"]
        pairs = sum(m * (m + 1) // 2 if case["causal"] else m * m for m in lengths)
        return {"bytes": 2 * sum(lengths) * (2 * h + 2 * kv) * dim, "flops": 4.0 * h * dim * pairs}
    if kind == "step":
        lengths, h, new = _lengths(case), case["heads"], case["new"]
        pairs = sum(new * (case["prefix"] + m) - new * (new - 1) // 2 for m in lengths)
        return {"bytes": 2 * (case["prefix"] + sum(lengths)) * 2 * kv * dim + 2 * 2 * case["seqs"] * new * h * dim,
                "flops": 4.0 * h * dim * pairs}
    token = 2 * 2 * case["layers"] * kv * dim
    n, tokens, new, page = case["seqs"], case["tokens"], case["new"], case["page"]
    if kind == "fork":
        tail = tokens % page
        # The tail read once and written for each sequence, the new tokens into the cache, all of it read back.
        return {"bytes": token * (tail + n * tail + 2 * n * new + 2 * n * (tail + new)), "flops": 0}
    return {"bytes": token * n * new * (2 + 2 + 2), "flops": 0}


def exact(case, seed):
    """The outputs in 64 bits, from the definition: sequence by sequence and head by head; copies as they are."""
    s = prepare(case, seed)
    kind, kv, dim = case["kind"], case["kv_heads"], case["dim"]
    if kind in ("fork", "compact"):
        n, new = case["seqs"], case["new"]
        parts = s["fresh"].double().unflatten(2, (n, new))
        if kind == "fork":
            tail = case["tokens"] % case["page"]
            kept = s["filled"][:, :, case["tokens"] - tail:].double()
            parts = torch.cat([kept[:, :, None].expand(-1, -1, n, -1, -1, -1), parts], dim=3)
        return parts.flatten(2, 3), None
    h = case["heads"]
    group, lengths = h // kv, _lengths(case)
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
        hide = None
        if kind == "step" or case["causal"]:
            hide = torch.ones(rows, k.shape[0], dtype=torch.bool, device="cuda").triu_(first + 1)
        for j in range(h):
            w = (q[:, j] @ k[:, j // group].T) / math.sqrt(dim)
            if hide is not None:
                w.masked_fill_(hide, -math.inf)
            o[:, j] = torch.softmax(w, dim=1) @ v[:, j // group]
    return out
