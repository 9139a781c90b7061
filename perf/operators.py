"""The operators of beam decoding, in their plain form and through the library.

Three operators work on the self K/V rows that the lanes of a batch keep:

* ``attend``: one new row per lane attends the rows of a prefix that several lanes share, the
  lane's own cached rows and itself, with an optional sliding window behind a few first rows that
  stay visible; the new K/V row is appended to the lane's cache.
* ``select``: of every request's beams x vocabulary continuations the best `beams` are picked by
  their summed log-probability.
* ``reorder``: the lanes' own rows follow the beams that were picked.

``run`` computes them with elementary torch operations, or, where ``own`` is set, through
libmynah_b200.so.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}

# ------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one stream at the position of the single-step benchmark: latency of the smallest call
        dict(name="attend one stream", op="attend", type="f32", lanes=1, heads=12, head_width=64, low=256, high=256,
             capacity=520, prefixes=0, prefix=0, window=0, sinks=0),
        # eight candidates of one request over its voice context
        dict(name="attend eight beams", op="attend", type="f32", lanes=8, heads=12, head_width=64, low=130, high=130,
             capacity=520, prefixes=1, prefix=217, window=0, sinks=0),
        # the serving batch: streams of different ages, four voices
        dict(name="attend sixty-four streams", op="attend", type="f32", lanes=64, heads=12, head_width=64, low=0, high=512,
             capacity=520, prefixes=4, prefix=217, window=0, sinks=0),
        # a large batch behind one long shared context, half-precision rows
        dict(name="attend long prefix", op="attend", type="f16", lanes=256, heads=12, head_width=64, low=0, high=500,
             capacity=520, prefixes=1, prefix=4096, window=0, sinks=0),
        # endless streams: a window behind four first rows, caches used as rings
        dict(name="attend window", op="attend", type="f16", lanes=48, heads=12, head_width=64, low=700, high=90001,
             capacity=1029, prefixes=0, prefix=0, window=1025, sinks=4),
        # few wide heads, long odd caches
        dict(name="attend wide heads", op="attend", type="f32", lanes=5, heads=3, head_width=128, low=1, high=9973,
             capacity=10007, prefixes=2, prefix=75, window=0, sinks=0),
        # one frame's table for one request
        dict(name="select one request", op="select", requests=1, beams=4, vocab=2048, codebook=2016, eos=2017),
        # the same for a serving batch
        dict(name="select sixty-four requests", op="select", requests=64, beams=8, vocab=2048, codebook=2016, eos=2017),
        # a text-sized vocabulary, odd, many beams
        dict(name="select large vocabulary", op="select", requests=24, beams=16, vocab=50021, codebook=50000, eos=50020),
        # a young request of two beams
        dict(name="reorder two beams", op="reorder", type="f32", requests=1, beams=2, layers=2, width=192, rows=24, capacity=96),
        # a serving batch of half-precision caches
        dict(name="reorder sixteen requests", op="reorder", type="f16", requests=16, beams=4, layers=12, width=768, rows=130,
             capacity=520),
        # whole 512-frame caches of every layer
        dict(name="reorder long caches", op="reorder", type="f32", requests=4, beams=8, layers=12, width=768, rows=512,
             capacity=520),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "select", "reorder"])
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = _log_int(rng, 64, 60000)
        requests = _log_int(rng, 1, max(1, min(256, 19_000_000 // (beams * vocab))))
        return dict(op=op, requests=requests, beams=beams, vocab=vocab, codebook=vocab - rng.randint(2, 40), eos=vocab - 1)
    kind = rng.choice(["f32", "f16"])
    size = 4 if kind == "f32" else 2
    if op == "reorder":
        beams = rng.randint(2, 16)
        width = 8 * rng.randint(4, 128)
        layers = rng.randint(1, 16)
        rows = _log_int(rng, 1, 1500)
        while 2 * layers * beams * rows * width * size > 1_000_000_000:
            rows = rows // 2
        requests = _log_int(rng, 1, max(1, min(64, 1_000_000_000 // (2 * layers * beams * rows * width * size))))
        return dict(op=op, type=kind, requests=requests, beams=beams, layers=layers, width=width, rows=rows,
                    capacity=rows + rng.randint(0, 40))
    head_width = rng.choice([16, 24, 32, 48, 64, 64, 64, 80, 96, 128, 128])
    heads = rng.randint(1, max(1, min(24, 1536 // head_width)))
    width = heads * head_width
    lanes = _log_int(rng, 1, 256)
    prefixes = rng.choice([0, 1, 1, 2, 5])
    prefix = _log_int(rng, 1, 4096) if prefixes else 0
    windowed = rng.random() < 0.4
    window, sinks = (_log_int(rng, 1, 2000), rng.randint(0, 16)) if windowed else (0, 0)
    high = _log_int(rng, 1, 60000)
    if not windowed:
        high = max(1, min(high, 350_000_000 // (lanes * width * size * 2)))
        capacity = high + 1 + rng.randint(0, 30)
    else:
        window = max(1, min(window, 350_000_000 // (lanes * width * size * 2)))
        capacity = window + sinks + rng.randint(0, 30)
    while lanes * prefix * width > 256 * 4096 * 768:
        prefix //= 2
    return dict(op=op, type=kind, lanes=lanes, heads=heads, head_width=head_width, low=rng.randint(0, high), high=high,
                capacity=capacity, prefixes=prefixes, prefix=prefix, window=window, sinks=sinks)


# ------------------------------------------------- what a case fixes: lengths, voices, parents


def _lengths(case):
    """Cached own rows of every lane, spread evenly over low .. high in a mixed order."""
    n, low, high = case["lanes"], case["low"], case["high"]
    got = [low + (high - low) * i // max(1, n - 1) for i in range(n)]
    random.Random(n).shuffle(got)
    return got


def _voices(case):
    """Prefix of every lane (one lane in sixteen has none where there are several) and their lengths."""
    p, r = case["prefixes"], random.Random(case["lanes"] + 1)
    lanes = [(p if p > 1 and r.randrange(16) == 0 else r.randrange(p)) if p else 0 for _ in range(case["lanes"])]
    return lanes, [max(0, case["prefix"] - 11 * i) for i in range(p)]


def _seen(length, prefix, window, sinks):
    """Ranges of prefix rows and of own rows (the new one, `length`, among them) that a lane sees."""
    if not window:
        return [(0, prefix)], [(0, length + 1)]
    first = prefix + length - window + 1                     # of the prefix and the own rows counted on
    head = min(sinks, max(0, first))
    return ([(0, min(head, prefix)), (min(max(first, 0), prefix), prefix)],
            [(0, max(0, head - prefix)), (max(0, first - prefix), length + 1)])


def _parents(case):
    r = random.Random(case["requests"] * 31 + case["beams"])
    return [[r.randrange(case["beams"]) for _ in range(case["beams"])] for _ in range(case["requests"])]


def _rows_of(case):
    """Own rows of every lane; the beams of one request are of one age."""
    n = case["requests"]
    return [max(1, case["rows"] - (case["rows"] // 3) * i // n) for i in range(n) for _ in range(case["beams"])]


def work(case):
    if case["op"] == "select":
        n = case["requests"] * case["beams"] * (case["codebook"] + 1)
        return {"bytes": 4 * n + 20 * case["requests"] * case["beams"], "flops": 4 * n}
    size = TYPES[case["type"]].itemsize
    if case["op"] == "reorder":
        moved, beams, rows = 0, case["beams"], _rows_of(case)
        for i, parents in enumerate(_parents(case)):
            pairs = [(b, p) for b, p in enumerate(parents) if b != p]
            moved += sum(rows[i * beams + p] for p in {p for _, p in pairs}) + sum(rows[i * beams + p] for _, p in pairs)
        return {"bytes": 2 * case["layers"] * case["width"] * size * moved, "flops": 0}
    width = case["heads"] * case["head_width"]
    voice, voice_rows = _voices(case)
    cached, seen, touched = 0, 0, [set() for _ in voice_rows]
    for length, v in zip(_lengths(case), voice):
        p = voice_rows[v] if v < len(voice_rows) else 0
        pre, mine = _seen(length, p, case["window"], case["sinks"])
        cached += sum(b - a for a, b in mine) - 1
        seen += sum(max(0, b - a) for a, b in pre + mine)
        if p:
            touched[v].update(x for x in pre if x[1] > x[0])
    shared = 0
    for ranges in touched:
        at = 0
        for a, b in sorted(ranges):
            shared += max(0, b - max(a, at))
            at = max(at, b)
    lanes = case["lanes"]
    return {"bytes": 2 * (cached + shared + lanes) * width * size + 4 * lanes * (4 * width + 3), "flops": 4 * width * seen}


# ------------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    s = {"case": dict(case)}
    if case["op"] == "select":
        n = case["requests"] * case["beams"]
        s["logits"] = 2.0 * normal(n, case["vocab"])
        s["score"] = -20.0 * torch.rand(n, generator=g, device=DEVICE)
        s["done"] = (torch.rand(n, generator=g, device=DEVICE) < 0.1).to(torch.int32)
        s["allow_eos"] = (torch.rand(case["requests"], generator=g, device=DEVICE) < 0.5).to(torch.int32)
        s["score_out"] = torch.empty(n, device=DEVICE)
        for name in ("token", "parent", "done_out"):
            s[name] = torch.empty(n, dtype=torch.int32, device=DEVICE)
        return s
    dtype = TYPES[case["type"]]
    if case["op"] == "reorder":
        n = case["requests"] * case["beams"]
        for name in ("k", "v"):
            s[name] = normal(n, case["layers"], case["capacity"], case["width"], dtype=dtype)
        s["parent"] = whole(sum(_parents(case), []))
        s["length"] = whole(_rows_of(case))
        s["length_out"] = torch.empty_like(s["length"])
        return s
    lanes, width = case["lanes"], case["heads"] * case["head_width"]
    s["qkv"] = normal(lanes, 3 * width)
    for name in ("k", "v"):
        s[name] = normal(lanes, case["capacity"], width, dtype=dtype)
        s["prefix_" + name] = normal(case["prefixes"], case["prefix"], width, dtype=dtype)
    voice, voice_rows = _voices(case)
    s["slot"] = torch.randperm(lanes, generator=g, device=DEVICE).to(torch.int32)
    s["length"], s["voice"], s["voice_rows"] = whole(_lengths(case)), whole(voice), whole(voice_rows)
    s["most"] = max(sum(b - a for a, b in _seen(n, voice_rows[v] if v < len(voice_rows) else 0, case["window"], case["sinks"])[1])
                    for n, v in zip(_lengths(case), voice))
    s["out"] = torch.empty(lanes, width, device=DEVICE)
    return s


# -------------------------------------------------------------------------------- plain forms


def _plain_select(s):
    c = s["case"]
    requests, beams, vocab = c["requests"], c["beams"], c["vocab"]
    token = torch.arange(vocab, device=DEVICE)
    allowed = (token < c["codebook"])[None, :] | ((token == c["eos"])[None, :] & (s["allow_eos"] != 0)[:, None])
    # 64 bits from here on: which of two close continuations is better is a border
    x = s["logits"].double().view(requests, beams, vocab).masked_fill(~allowed[:, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    done = (s["done"] != 0).view(requests, beams, 1)
    frozen = torch.where(token == c["eos"], 0.0, -math.inf).double()
    x = torch.where(done, frozen[None, None, :], x) + s["score"].double().view(requests, beams, 1)
    value, at = torch.sort(x.view(requests, beams * vocab), dim=-1, descending=True, stable=True)
    value, at = value[:, :beams], at[:, :beams]
    place = torch.arange(beams, device=DEVICE).expand(requests, beams)
    dead = value == -math.inf
    pick = torch.where(dead, 0, at % vocab)
    parent = torch.where(dead, place, at // vocab)
    return {"score": value.float().reshape(-1), "token": pick.to(torch.int32).reshape(-1),
            "parent": parent.to(torch.int32).reshape(-1),
            "done": ((pick == c["eos"]) & ~dead).to(torch.int32).reshape(-1)}


def _plain_reorder(s):
    c = s["case"]
    beams = c["beams"]
    lane = torch.arange(c["requests"] * beams, device=DEVICE)
    source = lane // beams * beams + s["parent"].long()
    rows = s["length"].long()[source]
    moved = (torch.arange(c["capacity"], device=DEVICE)[None, :] < rows[:, None])[:, None, :, None]
    for name in ("k", "v"):
        s[name].copy_(torch.where(moved, s[name][source], s[name]))
    s["length_out"].copy_(rows)
    return {"k": s["k"], "v": s["v"], "length": s["length_out"]}


def _plain_attend(s):
    c = s["case"]
    lanes, heads, hw, window, sinks = c["lanes"], c["heads"], c["head_width"], c["window"], c["sinks"]
    q, k, v = s["qkv"].view(lanes, 3, heads, hw).unbind(1)
    length, voice, slot = s["length"].long(), s["voice"].long(), s["slot"].long()
    if c["prefixes"]:
        rows = torch.where(voice < c["prefixes"], s["voice_rows"].long()[voice.clamp(max=c["prefixes"] - 1)], 0)
    else:
        rows = torch.zeros_like(length)
    keep = (sinks - rows).clamp(min=0)                       # own rows among the first ones that stay

    def place(r):                                            # row of the cache that own row r lies in
        k2 = keep if r.dim() == 1 else keep[:, None]
        return torch.where(r < k2, r, k2 + (r - k2).clamp(min=0) % (c["capacity"] - k2))

    s["k"][slot, place(length)] = k.reshape(lanes, -1).to(s["k"].dtype)
    s["v"][slot, place(length)] = v.reshape(lanes, -1).to(s["v"].dtype)
    # own rows that are seen: the first ones that stay, then the window up to the new row
    first = (length - window + 1).clamp(min=0) if window else torch.zeros_like(length)
    stay = torch.minimum(keep, first) if window else torch.zeros_like(length)
    i = torch.arange(s["most"], device=DEVICE)[None, :]
    r = torch.where(i < stay[:, None], i, first[:, None] + i - stay[:, None])
    seen = r <= length[:, None]
    at = place(torch.minimum(r, length[:, None]))
    mine_k = s["k"][slot[:, None], at].float().view(lanes, -1, heads, hw)
    mine_v = s["v"][slot[:, None], at].float().view(lanes, -1, heads, hw)
    scale = 1.0 / math.sqrt(hw)
    x = torch.einsum("lhd,lrhd->lhr", q, mine_k) * scale
    x = x.masked_fill(~seen[:, None, :], -math.inf)
    n = c["prefixes"] * c["prefix"]
    if n:
        j = torch.arange(c["prefix"], device=DEVICE)[None, None, :]
        p = torch.arange(c["prefixes"], device=DEVICE)[None, :, None]
        seen = (p == voice[:, None, None]) & (j < rows[:, None, None])
        if window:
            seen = seen & ((j < sinks) | (j > (rows + length - window)[:, None, None]))
        pre_k = s["prefix_k"].float().view(n, heads, hw)
        y = torch.einsum("lhd,jhd->lhj", q, pre_k) * scale
        x = torch.cat([y.masked_fill(~seen.view(lanes, 1, n), -math.inf), x], -1)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    out = torch.einsum("lhr,lrhd->lhd", x[..., n:], mine_v)
    if n:
        out = out + torch.einsum("lhj,jhd->lhd", x[..., :n], s["prefix_v"].float().view(n, heads, hw))
    s["out"].copy_(out.reshape(lanes, -1))
    return {"out": s["out"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------------------- through the library

_backend = None


def _library():
    """The backend a program keeps open, on torch's stream."""
    global _backend
    if _backend is None:
        from mynah_tts_b200.backend import Backend
        _backend = Backend("f32")
        _backend.set_stream(torch.cuda.current_stream().cuda_stream)
    return _backend


def _bound(s):
    """The call as a decode loop keeps it: its descriptor is filled once."""
    b, c = _library(), s["case"]
    at = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor) and v.numel()}
    if c["op"] == "select":
        return b.bind_beam_select(
            logits=at["logits"], requests=c["requests"], beams=c["beams"], vocab=c["vocab"], codebook_size=c["codebook"],
            eos_id=c["eos"], allow_eos=at["allow_eos"], score=at["score"], done=at["done"], score_out=at["score_out"],
            token=at["token"], parent=at["parent"], done_out=at["done_out"])
    if c["op"] == "reorder":
        cache = b.lane_cache(c["type"], at["k"], at["v"], slots=c["requests"] * c["beams"], capacity=c["capacity"],
                             width=c["width"], slot_stride=c["layers"] * c["capacity"] * c["width"], layers=c["layers"],
                             layer_stride=c["capacity"] * c["width"])
        return b.bind_beam_reorder(cache, requests=c["requests"], beams=c["beams"], parent=at["parent"], length=at["length"],
                                   length_out=at["length_out"])
    width = c["heads"] * c["head_width"]
    cache = b.lane_cache(c["type"], at["k"], at["v"], slots=c["lanes"], capacity=c["capacity"], width=width)
    more = {}
    if "prefix_k" in at:
        more = dict(prefix_k=at["prefix_k"], prefix_v=at["prefix_v"], prefixes=c["prefixes"], prefix_capacity=c["prefix"],
                    prefix_length=at["voice_rows"], lane_prefix=at["voice"])
    n = b.lane_attention_workspace(c["lanes"], c["heads"], c["head_width"], c["prefixes"] if more else 0,
                                   c["prefix"] if more else 0)
    s["workspace"] = torch.empty(n, device=DEVICE)
    return b.bind_lane_attention(
        cache, lanes=c["lanes"], heads=c["heads"], head_width=c["head_width"], scale=1.0 / math.sqrt(c["head_width"]),
        qkv=at["qkv"], length=at["length"], slot=at["slot"], window=c["window"], sinks=c["sinks"], out=at["out"],
        workspace=s["workspace"].data_ptr(), workspace_floats=n, **more)


def run(state):
    op = state["case"]["op"]
    if own:
        if "call" not in state:
            state["call"] = _bound(state)
        state["call"]()
        if op == "select":
            return {"score": state["score_out"], "token": state["token"], "parent": state["parent"], "done": state["done_out"]}
        if op == "reorder":
            return {"k": state["k"], "v": state["v"], "length": state["length_out"]}
        return {"out": state["out"], "k": state["k"], "v": state["v"]}
    return {"select": _plain_select, "reorder": _plain_reorder, "attend": _plain_attend}[op](state)


# -------------------------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(case, s)
    if case["op"] == "reorder":
        k, v, beams = s["k"].double(), s["v"].double(), case["beams"]
        rows = _rows_of(case)
        for i, parents in enumerate(_parents(case)):
            for b, p in enumerate(parents):
                n = rows[i * beams + p]
                k[i * beams + b, :, :n] = s["k"][i * beams + p, :, :n].double()
                v[i * beams + b, :, :n] = s["v"][i * beams + p, :, :n].double()
        return {"k": k, "v": v, "length": None}
    return _exact_attend(case, s)


def _exact_select(case, s):
    beams, best = case["beams"], []
    logits, score = s["logits"].double(), s["score"].double()
    done, allow = s["done"].tolist(), s["allow_eos"].tolist()
    for i in range(case["requests"]):
        per_beam = []
        for b in range(beams):
            lane = i * beams + b
            if done[lane]:
                per_beam.append(score[lane:lane + 1])
                continue
            row = logits[lane, :case["codebook"]]
            if allow[i]:
                row = torch.cat([row, logits[lane, case["eos"]:case["eos"] + 1]])
            per_beam.append(torch.topk(torch.log_softmax(row, 0) + score[lane], min(beams, row.numel())).values)
        top = torch.sort(torch.cat(per_beam), descending=True).values[:beams]
        best.append(torch.cat([top, torch.full((beams - top.numel(),), -math.inf, dtype=torch.float64, device=DEVICE)]))
    return {"score": torch.cat(best), "token": None, "parent": None, "done": None}


def _exact_attend(case, s):
    lanes, heads, hw = case["lanes"], case["heads"], case["head_width"]
    voice, voice_rows = _voices(case)
    slots, dtype = s["slot"].tolist(), s["k"].dtype
    k, v = s["k"].double(), s["v"].double()
    q = s["qkv"].double().view(lanes, 3, heads, hw)
    out = torch.empty(lanes, heads * hw, dtype=torch.float64, device=DEVICE)
    for lane, length in enumerate(_lengths(case)):
        p = voice_rows[voice[lane]] if voice[lane] < len(voice_rows) else 0
        keep = max(0, case["sinks"] - p)
        pre, mine = _seen(length, p, case["window"], case["sinks"])

        def place(r):
            return r if r < keep else keep + (r - keep) % (case["capacity"] - keep)
        slot = slots[lane]
        k[slot, place(length)] = q[lane, 1].reshape(-1).to(torch.float32).to(dtype).double()
        v[slot, place(length)] = q[lane, 2].reshape(-1).to(torch.float32).to(dtype).double()
        rows = torch.tensor([place(r) for a, b in mine for r in range(a, b)], device=DEVICE)
        ks, vs = [k[slot, rows]], [v[slot, rows]]
        for a, b in pre:
            if b > a:
                ks.append(s["prefix_k"][voice[lane], a:b].double())
                vs.append(s["prefix_v"][voice[lane], a:b].double())
        kk, vv = torch.cat(ks).view(-1, heads, hw), torch.cat(vs).view(-1, heads, hw)
        w = torch.softmax((kk * q[lane, 0]).sum(-1) / math.sqrt(hw), 0)
        out[lane] = (w[..., None] * vv).sum(0).reshape(-1)
    return {"out": out, "k": k, "v": v}
