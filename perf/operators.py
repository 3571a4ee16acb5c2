"""The operators of a program that keeps its own model loop and serves several sequences from a paged cache: rotary positions
of many tokens, attention over whole prompts, attention of new tokens over the cache (kuiperllama_amd.ops).

Kinds of cases:

  "store"   rope_store: the queries of a batch of tokens rotated, its keys rotated and written with its values into the pages
  "rotate"  rope_tokens: queries and keys rotated, out of rows that hold q, k and v side by side
  "packed"  attn_packed: causal attention of whole prompts of different lengths, one behind the other
  "paged"   attn_paged: `new` tokens of each sequence over the `lens` keys that its pages hold

A query head h reads key head h // (heads / kv_heads).  Pages lie in the cache in an order of their own.
"""
import math
import random

import torch

own = False  # False: the plain forms below; True: the framework's operators

_HALF, _INTERLEAVED = "half", "interleaved"


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _spread(seed, n, low, high):
    """n lengths between low and high, evenly over their logarithm."""
    r = random.Random(seed)
    return [int(round(math.exp(r.uniform(math.log(low), math.log(high))))) for _ in range(n)]


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded token of each of 48 chats, far into their contexts, frequencies scaled in bands: nothing but latency
        {"name": "store-step-48", "kind": "store", "dtype": "bf16", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 64, "rot": 64,
         "mode": _HALF, "theta": 500000.0, "scaling": "bands", "factor": 32.0, "page": 16, "far": 131072},
        # a full pass of prompt tokens of a model whose heads all have keys of their own: bandwidth
        {"name": "store-prompts-8192", "kind": "store", "dtype": "bf16", "tokens": 8192, "heads": 32, "kv_heads": 32, "dim": 128,
         "rot": 128, "mode": _HALF, "theta": 10000.0, "scaling": "linear", "factor": 4.0, "page": 64, "far": 16384},
        # a ragged prompt in fp32, half of the head rotated, by pairs of neighbours, out of rows of q, k and v
        {"name": "rotate-part-1901", "kind": "rotate", "dtype": "fp32", "tokens": 1901, "heads": 32, "kv_heads": 4, "dim": 64, "rot": 32,
         "mode": _INTERLEAVED, "theta": 10000.0, "scaling": "ramp", "factor": 40.0, "far": 65536},
        # three short questions in fp32: latency
        {"name": "packed-short-fp32", "kind": "packed", "dtype": "fp32", "heads": 14, "kv_heads": 2, "dim": 64, "lens": "7,33,1", "window": 0},
        # the prompts of an ordinary batch, from a few tokens to a long document
        {"name": "packed-ragged-20", "kind": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 64,
         "lens": _text(_spread(7, 20, 9, 4000)), "window": 0},
        # one very long document: matrix products and exponentials
        {"name": "packed-long-16384", "kind": "packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "lens": "16384", "window": 0},
        # prompts of an fp32 model, a key head for each query head
        {"name": "packed-fp32-4", "kind": "packed", "dtype": "fp32", "heads": 32, "kv_heads": 32, "dim": 128, "lens": "2048,777,512,130",
         "window": 0},
        # the next token of one sequence that fills its context: the whole chip on one row of queries
        {"name": "paged-step-131072", "kind": "paged", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 64, "new": "1", "lens": "131072",
         "window": 0, "page": 256},
        # the next token of 64 sequences of very different lengths
        {"name": "paged-step-64", "kind": "paged", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "new": _text([1] * 64),
         "lens": _text(_spread(11, 64, 90, 8192)), "window": 0, "page": 64},
        # the next token of a few short chats in fp32: latency
        {"name": "paged-step-fp32-8", "kind": "paged", "dtype": "fp32", "heads": 14, "kv_heads": 2, "dim": 64, "new": _text([1] * 8),
         "lens": _text(_spread(13, 8, 17, 700)), "window": 0, "page": 16},
        # a portion of a long prompt behind what the cache already holds of it
        {"name": "paged-chunk-512", "kind": "paged", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "new": "512", "lens": "32768",
         "window": 0, "page": 128},
        # portions of two prompts among 30 decoded tokens, a sliding window, pages of an odd size
        {"name": "paged-mixed-32", "kind": "paged", "dtype": "bf16", "heads": 32, "kv_heads": 4, "dim": 64,
         "new": _text([300] + [1] * 20 + [77] + [1] * 10), "lens": _text([2100] + _spread(17, 20, 30, 6000) + [77] + _spread(19, 10, 30, 6000)),
         "window": 1024, "page": 48},
    ]


_MOST_FLOPS = {"bf16": 2.0e12, "fp32": 2.0e11}  # of a drawn case: below the time of the largest listed ones
_MOST_BYTES = 5.0e8


def draw(rng):
    def log(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    while True:
        heads, kv_heads = rng.choice([(32, 8), (32, 4), (14, 2), (32, 32), (6, 6), (16, 4), (12, 1)])
        dim = rng.choice([48, 64, 64, 80, 128, 128, 256])
        case = {"kind": rng.choice(["store", "rotate", "packed", "packed", "paged", "paged", "paged"]),
                "dtype": rng.choice(["bf16", "bf16", "fp32"]), "heads": heads, "kv_heads": kv_heads, "dim": dim}
        if case["kind"] in ("store", "rotate"):
            rot = rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2])
            case.update(tokens=log(1, 8192), rot=rot, mode=rng.choice([_HALF, _INTERLEAVED]), theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                        scaling=rng.choice(["none", "linear", "bands", "ramp"]), factor=rng.choice([2.0, 8.0, 40.0]),
                        far=log(4096, 1 << 20))
            if case["kind"] == "store":
                case["page"] = rng.choice([1, 16, 24, 64, 256])
        else:
            case["window"] = rng.choice([0, 0, 0, log(1, 4096)])
            if case["kind"] == "packed":
                longest = log(8, 16384)
                case["lens"] = _text(log(max(1, longest // 64), longest) for _ in range(log(1, 32)))
            else:
                case["page"] = rng.choice([16, 16, 48, 64, 100, 256])
                longest, most = log(16, 131072), rng.choice([1, 1, 4, log(1, 1024)])
                lens = [log(max(1, longest // 64), longest) for _ in range(log(1, 128))]
                case["lens"] = _text(lens)
                case["new"] = _text(min(n, log(1, most)) for n in lens)
        w = work(case)
        if w["flops"] <= _MOST_FLOPS[case["dtype"]] and w["bytes"] <= _MOST_BYTES:
            return case


# ---- their work --------------------------------------------------------------------------------------------------------
def _size(case):
    return 2 if case["dtype"] == "bf16" else 4


def _sequences(case):
    """(new tokens, keys) of each sequence."""
    lens = _numbers(case["lens"])
    return list(zip(_numbers(case["new"]) if case["kind"] == "paged" else lens, lens))


def _pairs(new, length, window):
    """Pairs of a query and a key that it sees, and the keys that any of them sees."""
    if window <= 0 or window >= length:
        return new * (length - new) + new * (new + 1) // 2, length
    full = max(0, min(new, length - window + 1))  # queries at places >= window - 1
    rest = new - full
    return full * window + rest * (length - new) + rest * (rest + 1) // 2, min(length, new + window - 1)


def work(case):
    row = (case["heads"] + case["kv_heads"]) * case["dim"] * _size(case)
    if case["kind"] in ("store", "rotate"):
        values = case["kv_heads"] * case["dim"] * _size(case) if case["kind"] == "store" else 0
        return {"bytes": case["tokens"] * 2 * (row + values), "flops": case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"] * 3}
    queries = pairs = keys = 0
    for new, length in _sequences(case):
        p, k = _pairs(new, length, case["window"])
        queries, pairs, keys = queries + new, pairs + p, keys + k
    return {"bytes": (2 * queries * case["heads"] + 2 * keys * case["kv_heads"]) * case["dim"] * _size(case),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _random(gen, case, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(_type(case))


def _scaling(case):
    """As the config.json of a model says it."""
    f = case["factor"]
    return {"none": None, "linear": {"rope_type": "linear", "factor": f},
            "bands": {"rope_type": "llama3", "factor": f, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                      "original_max_position_embeddings": 8192},
            "ramp": {"rope_type": "yarn", "factor": f, "beta_fast": 32.0, "beta_slow": 1.0,
                     "original_max_position_embeddings": 4096}}[case["scaling"]]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, KH, D = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["kind"] in ("store", "rotate"):
        T = case["tokens"]
        rows = _random(gen, case, T, (H + 2 * KH) * D)  # what the three projections of a layer leave
        s["q"] = rows[:, :H * D].view(T, H, D)
        s["k"] = rows[:, H * D:(H + KH) * D].view(T, KH, D)
        s["v"] = rows[:, (H + KH) * D:].view(T, KH, D)
        s["positions"] = torch.randint(0, case["far"], (T,), device="cuda", generator=gen, dtype=torch.int32)
        s["q_out"] = torch.zeros(T, H, D, device="cuda", dtype=_type(case))
        if case["kind"] == "rotate":
            s["k_out"] = torch.zeros(T, KH, D, device="cuda", dtype=_type(case))
        else:
            pages = T // case["page"] + 3
            s["kcache"] = _random(gen, case, pages, case["page"], KH, D)
            s["vcache"] = _random(gen, case, pages, case["page"], KH, D)
            s["slots"] = torch.randperm(pages * case["page"], device="cuda", generator=gen)[:T].to(torch.int32)
        return s
    seqs = _sequences(case)
    T, B = sum(n for n, _ in seqs), len(seqs)
    s["q"] = _random(gen, case, T, H, D, scale=2.0)  # scores of a spread of 2: some keys count, most hardly do
    ends = [0]
    for n, _ in seqs:
        ends.append(ends[-1] + n)
    s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    s["out"] = torch.zeros(T, H, D, device="cuda", dtype=_type(case))
    if case["kind"] == "packed":
        s["k"], s["v"] = _random(gen, case, T, KH, D), _random(gen, case, T, KH, D)
        return s
    held = [-(-length // case["page"]) for _, length in seqs]
    pages = sum(held) + 5
    s["kcache"] = _random(gen, case, pages, case["page"], KH, D)
    s["vcache"] = _random(gen, case, pages, case["page"], KH, D)
    order = torch.randperm(pages, device="cuda", generator=gen)[:sum(held)].to(torch.int32)
    table = torch.zeros(B, max(held), dtype=torch.int32, device="cuda")
    for b, part in enumerate(order.split(held)):
        table[b, :held[b]] = part
    s["pages"] = table
    s["lengths"] = torch.tensor([length for _, length in seqs], dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handles that a program keeps: a table of frequencies, a workspace
        from kuiperllama_amd import ops
        if case["kind"] in ("store", "rotate"):
            s["table"] = ops.rope_table(case["rot"], case["theta"], device="cuda", scaling=_scaling(case))
            s["mode"] = ops.ROPE_HALF if case["mode"] == _HALF else ops.ROPE_INTERLEAVED
        elif case["kind"] == "paged":
            s["workspace"] = ops.attn_paged_workspace(case["heads"], case["kv_heads"], case["dim"], s["q"].shape[0], s["q"].device)
            s["max_new"] = max(n for n, _ in _sequences(case))
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians a position of each pair, in 64 bits, and the factor of a rotated pair's length."""
    i = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
    f = case["theta"] ** (-2.0 * i / case["rot"])
    c = _scaling(case)
    if c is None:
        return f, 1.0
    if c["rope_type"] == "linear":
        return f / c["factor"], 1.0
    original = c["original_max_position_embeddings"]
    if c["rope_type"] == "llama3":
        turns, low, high = original * f / (2 * math.pi), c["low_freq_factor"], c["high_freq_factor"]
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return f * keep + f / c["factor"] * (1 - keep), 1.0

    def pair(turns):
        return case["rot"] * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))

    low, high = max(math.floor(pair(c["beta_fast"])), 0), min(math.ceil(pair(c["beta_slow"])), case["rot"] - 1)
    ramp = ((i - low) / (max(high - low, 0.001))).clamp(0.0, 1.0)
    return f / c["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(c["factor"]) + 1.0


def _rotate(case, x, positions, freqs, magnitude):
    angle = positions.double()[:, None] * freqs
    cos, sin = (angle.cos() * magnitude).float()[:, None, :], (angle.sin() * magnitude).float()[:, None, :]
    rot, y = case["rot"], x.float()
    out = y.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if case["mode"] == _HALF else (slice(0, rot, 2), slice(1, rot, 2))
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., a] * sin + y[..., b] * cos
    return out.to(x.dtype)


def _attend(q, k, v, window):
    """n queries at the last n places of the keys; [n, heads, dim], [keys, kv_heads, dim]."""
    n, heads, dim = q.shape
    keys, kv = k.shape[:2]
    kt, vt = k.float().permute(1, 2, 0).contiguous(), v.float().permute(1, 0, 2).contiguous()
    out = torch.empty(n, heads, dim, dtype=q.dtype, device=q.device)
    step = max(1, (1 << 28) // (heads * keys))
    for i in range(0, n, step):
        qs = q[i:i + step].float()
        m = qs.shape[0]
        qs = qs.view(m, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        s = torch.matmul(qs, kt).view(kv, heads // kv, m, keys) * dim ** -0.5
        place = torch.arange(keys - n + i, keys - n + i + m, device=q.device)[:, None]
        j = torch.arange(keys, device=q.device)[None, :]
        hidden = j > place
        if window > 0:
            hidden = hidden | (j <= place - window)
        s.masked_fill_(hidden, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p.view(kv, -1, keys), vt).view(kv, heads // kv, m, dim) / p.sum(-1, keepdim=True)
        out[i:i + step] = o.permute(2, 0, 1, 3).reshape(m, heads, dim).to(q.dtype)
    return out


def _plain(s):
    case = s["case"]
    if case["kind"] in ("store", "rotate"):
        freqs, magnitude = _frequencies(case)
        s["q_out"].copy_(_rotate(case, s["q"], s["positions"], freqs, magnitude))
        k = _rotate(case, s["k"], s["positions"], freqs, magnitude)
        if case["kind"] == "rotate":
            s["k_out"].copy_(k)
            return s["q_out"], s["k_out"]
        slots = s["slots"].long()
        s["kcache"].view(-1, *k.shape[1:])[slots] = k
        s["vcache"].view(-1, *k.shape[1:])[slots] = s["v"]
        return s["q_out"], s["kcache"], s["vcache"]
    first = 0
    for b, (new, length) in enumerate(_sequences(case)):
        rows = slice(first, first + new)
        if case["kind"] == "packed":
            k, v = s["k"][rows], s["v"][rows]
        else:
            held = s["pages"][b, :-(-length // case["page"])].long()
            k, v = (s[c][held].flatten(0, 1)[:length] for c in ("kcache", "vcache"))
        s["out"][rows] = _attend(s["q"][rows], k, v, case["window"])
        first += new
    return s["out"]


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from kuiperllama_amd import ops
    s, case = state, state["case"]
    if case["kind"] == "store":
        ops.rope_store(s["q"], s["k"], s["v"], s["positions"], s["table"], s["mode"], s["kcache"], s["vcache"], s["slots"], q_out=s["q_out"])
        return s["q_out"], s["kcache"], s["vcache"]
    if case["kind"] == "rotate":
        ops.rope_tokens(s["q"], s["k"], s["positions"], s["table"], s["mode"], q_out=s["q_out"], k_out=s["k_out"])
        return s["q_out"], s["k_out"]
    if case["kind"] == "packed":
        return ops.attn_packed(s["q"], s["k"], s["v"], s["offsets"], s["out"], window=case["window"])
    return ops.attn_paged(s["q"], s["kcache"], s["vcache"], s["pages"], s["lengths"], s["offsets"], s["out"], s["workspace"],
                          window=case["window"], max_new=s["max_new"])


# ---- from the definition, in 64 bits -------------------------------------------------------------------------------------
def _turned(case, x, positions):
    """Pairs as complex numbers times magnitude * exp(i * angle)."""
    radians, length, rot = [], 1.0, case["rot"]
    for i in range(rot // 2):
        f = 1.0 / case["theta"] ** (2 * i / rot)
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "bands":  # whole below 1/4 of the old context a wave, stretched beyond all of it
            wave = 2 * math.pi / f
            if wave > 8192 / 1.0:
                f /= case["factor"]
            elif wave >= 8192 / 4.0:
                part = (8192 / wave - 1.0) / (4.0 - 1.0)
                f = (1 - part) * f / case["factor"] + part * f
        elif case["scaling"] == "ramp":  # pairs that turn 32 times in the old context stay, those below one turn are stretched
            at = [rot * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(case["theta"])) for turns in (32.0, 1.0)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            part = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = part * f / case["factor"] + (1 - part) * f
            length = 1.0 + math.log(case["factor"]) / 10.0
        radians.append(f)
    angle = torch.outer(positions.double(), torch.tensor(radians, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(angle, length), angle)[:, None, :]
    y = x.double()
    part = y[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2) if case["mode"] == _HALF else y[..., :rot].unflatten(-1, (-1, 2))
    part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    part = part.transpose(-1, -2).flatten(-2) if case["mode"] == _HALF else part.flatten(-2)
    return torch.cat([part, y[..., rot:]], -1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("store", "rotate"):
        q, k = _turned(case, s["q"], s["positions"]), _turned(case, s["k"], s["positions"])
        if case["kind"] == "rotate":
            return q, k
        kc, vc = s["kcache"].double(), s["vcache"].double()
        at = (s["slots"].long() // case["page"], s["slots"].long() % case["page"])
        kc[at], vc[at] = k, s["v"].double()
        return q, kc, vc
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    last = 0
    for b, (new, length) in enumerate(_sequences(case)):
        last += new
        place = torch.arange(length, device="cuda")
        if case["kind"] == "paged":
            slot = s["pages"][b].long()[place // case["page"]] * case["page"] + place % case["page"]
            keys, values = s["kcache"].flatten(0, 1)[slot], s["vcache"].flatten(0, 1)[slot]
        else:
            keys, values = s["k"][last - length:last], s["v"][last - length:last]
        for h in range(case["heads"]):
            k, v = keys[:, h // group].double(), values[:, h // group].double()
            for first in range(0, new, 4096):
                i = torch.arange(first, min(new, first + 4096), device="cuda")
                score = s["q"][last - new + i, h].double() @ k.t() / math.sqrt(case["dim"])
                behind = (length - new + i)[:, None] - place[None, :]  # how far the key lies back
                seen = behind >= 0
                if case["window"] > 0:
                    seen &= behind < case["window"]
                out[last - new + i, h] = torch.softmax(score.masked_fill(~seen, -math.inf), -1) @ v
    return out
