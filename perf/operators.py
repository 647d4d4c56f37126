"""What a prompt that arrives in portions costs at the text tower's cache: three operators, as cases that can be timed and checked.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass through an operator
(in elementary torch operations, or with `own` through the framework's entry points), `exact` is the same in 64 bits.

  turn    `ops.qk_norm_rope`: RMS norm of every query and key head and the rotation by position in one pass, straight from the
          rows of a QKV product; halves or interleaved pairs, the whole head or its first part, frequencies stretched or not
  append  `ops.qkv_norm_rope_append_portions`: the same for the rows of a step that bring several sequences' next tokens, which
          also puts their keys and values into a paged cache
  attend  `ops.gqa_attention_portions_paged`: causal attention of those rows over the paged cache that holds them

A sequence's rows stand together; sequence b has the rows row_start[b] .. row_start[b + 1] - 1, and they are the last tokens of
its seq_lens[b].  Pages lie scattered, as an arena that has served other sequences hands them out.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
THETA = 1e6
SECTIONS = (24, 20, 20)  # of the three position axes, in pairs


# ---- the cases ------------------------------------------------------------------------------------------------------------

def _turn(name, **kw):
    return dict(dict(name=name, kind="turn", dtype="f16", rows=1, hq=16, hkv=8, d=128, rot=128, interleaved=False, norm=True, axes=1,
                     stretch=1.0, reach=32768), **kw)


def _append(name, **kw):
    return dict(dict(name=name, kind="append", dtype="f16", batch=1, rows_lo=1, rows_hi=1, cached_lo=0, cached_hi=0, hq=16, hkv=8,
                     d=128, rot=128, interleaved=False, norm=True, axes=1, page=64, first=False), **kw)


def _attend(name, **kw):
    return dict(dict(name=name, kind="attend", dtype="f16", batch=1, rows_lo=1, rows_hi=1, cached_lo=0, cached_hi=0, hq=16, hkv=8,
                     d=128, window=0, page=64), **kw)


def listed():
    return [
        # a few decoded tokens of a model with interleaved pairs, in the language models' type: latency
        _turn("turn_token_bf16", dtype="bf16", rows=8, hq=32, interleaved=True),
        # a long prompt of the tower, positions on three axes
        _turn("turn_prompt_f16", rows=8192, axes=3),
        # an odd prompt in the reference's type: a small model that turns only half of each head, stretched to four times its context
        _turn("turn_part_f32", dtype="f32", rows=1435, hq=12, hkv=4, d=80, rot=40, norm=False, stretch=4.0, reach=131072),
        # one token for each of a batch's sequences, the first layer of a step, which also advances the lengths
        _append("append_tokens_f16", batch=8, cached_lo=500, cached_hi=2040, first=True),
        # a step's token budget of portions from four prompts, in the middle of them
        _append("append_portions_f16", batch=4, rows_lo=200, rows_hi=1200, cached_lo=1, cached_hi=6000, axes=3),
        # two prompts from their beginning in the reference's type, large pages
        _append("append_prompts_f32", dtype="f32", batch=2, rows_lo=333, rows_hi=777, hq=12, hkv=4, d=64, rot=32, norm=False,
                interleaved=True, page=128),
        # a follow-up question in a short chat: latency
        _attend("attend_turn_f16", rows_lo=13, rows_hi=13, cached_lo=700, cached_hi=700),
        # a handful of drafted tokens for each of eight long conversations: reading the cache
        _attend("attend_drafts_f16", batch=8, rows_lo=1, rows_hi=8, cached_lo=9000, cached_hi=30000),
        # a step's token budget of one long prompt, its last portion
        _attend("attend_portion_f16", rows_lo=2048, rows_hi=2048, cached_lo=14000, cached_hi=14000),
        # whole prompts of unequal length side by side: the products
        _attend("attend_prompts_f16", batch=4, rows_lo=1500, rows_hi=8000),
        # a model with heads of 64, three queries to a key, and a sliding window
        _attend("attend_window_f16", batch=3, rows_lo=700, rows_hi=1900, cached_lo=100, cached_hi=9000, hq=24, hkv=8, d=64,
                window=2048),
        # portions in the reference's type
        _attend("attend_portions_f32", dtype="f32", batch=2, rows_lo=150, rows_hi=600, cached_lo=1000, cached_hi=3000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["turn", "append", "attend", "attend", "attend"])
    hkv = rng.choice([1, 2, 4, 8])
    heads = dict(hq=hkv * rng.choice([1, 2, 3, 4, 6, 8]), hkv=hkv)
    if kind == "turn":
        d = rng.choice([64, 80, 96, 128, 256])
        return dict(_turn("", dtype=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 1, 3000), d=d, axes=rng.choice([1, 3]),
                          rot=rng.choice([d, d // 2]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.7,
                          stretch=rng.choice([1.0, 2.0, 8.0]), reach=_log(rng, 1000, 500000)), **heads, name=None)
    batch = _log(rng, 1, 12)
    if kind == "append":
        d = rng.choice([64, 80, 96, 128, 256])
        rows = _log(rng, 1, 3000 // batch)
        return dict(_append("", dtype=rng.choice(["f16", "f16", "f32"]), batch=batch, rows_lo=rng.randint(1, rows), rows_hi=rows, d=d,
                            cached_hi=_log(rng, 1, 4000), rot=rng.choice([d, d // 2]), interleaved=rng.random() < 0.5,
                            norm=rng.random() < 0.7, axes=rng.choice([1, 3]), page=rng.choice([64, 128]),
                            first=rng.random() < 0.5), **heads, name=None)
    f32 = rng.random() < 0.2
    rows = _log(rng, 1, (600 if f32 else 4000) // batch)
    cached = _log(rng, 1, (4000 if f32 else 24000))
    case = dict(_attend("", dtype="f32" if f32 else "f16", batch=batch, rows_lo=rng.randint(1, rows), rows_hi=rows,
                        cached_lo=rng.randint(0, cached), cached_hi=cached, d=rng.choice([64, 80, 96, 128]),
                        window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]), page=rng.choice([64, 128])), **heads, name=None)
    while work(case)["flops"] > 5e11:
        case["rows_lo"], case["rows_hi"] = (case["rows_lo"] + 1) // 2, (case["rows_hi"] + 1) // 2
    return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, unequal and in no order."""
    return [int(round(hi - (hi - lo) * ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _counts(case):
    """(rows, tokens cached before them) of every sequence."""
    return list(zip(_spread(case["rows_lo"], case["rows_hi"], case["batch"]),
                    reversed(_spread(case["cached_lo"], case["cached_hi"], case["batch"]))))


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _frequencies(case):
    """theta^(-2i/rot), positions stretched over the context the model was trained on, and the factor of sine and cosine."""
    rot, stretch = case["rot"], case.get("stretch", 1.0)
    freq = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot) / stretch
    return freq.to(DEV), 0.1 * math.log(stretch) + 1.0


def _weights(case, dtype, gen):
    if not case["norm"]:
        return None, None
    return tuple((1 + 0.1 * torch.randn(case["d"], generator=gen, device=DEV)).to(dtype) for _ in range(2))


def _cache(case, counts, dtype, gen):
    """Pools of scattered pages, the block table and the lengths (new tokens included)."""
    page, lens = case["page"], [n + cached for n, cached in counts]
    blocks = [-(-n // page) for n in lens]
    total = sum(blocks) + 3
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), max(blocks)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, case["hkv"], page, case["d"])
    pools = [torch.randn(shape, generator=gen, device=DEV).to(dtype) for _ in range(2)]
    return pools, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, d, hq, hkv = DTYPES[case["dtype"]], case["d"], case["hq"], case["hkv"]
    s = dict(case=case)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=DEV).to(dtype)  # noqa: E731
    if case["kind"] == "turn":
        rows = case["rows"]
        s["qkv"] = randn(rows, (hq + 2 * hkv) * d)
        s["q"] = s["qkv"][:, :hq * d].view(rows, hq, d)
        s["k"] = s["qkv"][:, hq * d:(hq + hkv) * d].view(rows, hkv, d)
        shape = (rows,) if case["axes"] == 1 else (3, rows)
        s["pos"] = torch.randint(0, case["reach"], shape, generator=gen, device=DEV)
    else:
        counts = _counts(case)
        rows = sum(n for n, _ in counts)
        starts = [0]
        for n, _ in counts:
            starts.append(starts[-1] + n)
        s["row_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        (s["k_pages"], s["v_pages"]), s["table"], s["lens"] = _cache(case, counts, dtype, gen)
        if case["kind"] == "attend":
            s["q"] = (1.5 * torch.randn((rows, hq, d), generator=gen, device=DEV)).to(dtype)
            s["longest"] = max(n + cached for n, cached in counts)
            return s
        s["qkv"] = randn(rows, (hq + 2 * hkv) * d)
        s["pos"] = None
        if case["axes"] == 3:  # rows of an image stand at one time, columns and lines apart
            pos = torch.cat([torch.arange(cached, cached + n) for n, cached in counts]).to(DEV)
            s["pos"] = torch.stack([pos // 7, pos // 3, pos])
        s["before"] = s["lens"] - torch.tensor([n for n, _ in counts], dtype=torch.int32, device=DEV)
    s["freq"], s["factor"] = _frequencies(case)
    s["q_weight"], s["k_weight"] = _weights(case, dtype, gen)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------

def _axis_of_pair(pairs):
    """The position axis of each pair: the stride-3 rule of the tower."""
    i = torch.arange(pairs, device=DEV)
    axis = torch.zeros_like(i)
    axis[(i % 3 == 1) & (i < 3 * SECTIONS[1])] = 1
    axis[(i % 3 == 2) & (i < 3 * SECTIONS[2])] = 2
    return axis


def _plain_turn(x, weight, pos, freq, factor, interleaved):
    """x (rows, heads, d): the norm of every head, then the rotation of its first elements; in 32 bits, angles in 64."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    rot = 2 * freq.numel()
    at = pos.double()[:, None] if pos.dim() == 1 else pos.double()[_axis_of_pair(freq.numel())].T
    angle = at * freq
    c, s = (factor * torch.cos(angle)).float()[:, None], (factor * torch.sin(angle)).float()[:, None]
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _slots(s):
    """Of every row: its sequence's page at its position, the place in that page, and the position."""
    row_start, lens, page = s["row_start"].long(), s["lens"].long(), s["case"]["page"]
    rows = torch.arange(s["qkv"].shape[0], device=DEV)
    seq = torch.searchsorted(row_start, rows, right=True) - 1
    at = lens[seq] - row_start[seq + 1] + rows
    return s["table"][seq, at // page].long(), at % page, at


def _run_turn(s):
    case = s["case"]
    if own:
        from axono_b200 import ops

        return ops.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], s["q_weight"], s["k_weight"], EPS, interleaved=case["interleaved"],
                                factor=s["factor"], mrope_section=SECTIONS if case["axes"] == 3 else None)
    return tuple(_plain_turn(x, w, s["pos"], s["freq"], s["factor"], case["interleaved"])
                 for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _run_append(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = s["before"].clone() if case["first"] else s["lens"]
    if own:
        from axono_b200 import ops

        q = ops.qkv_norm_rope_append_portions(s["qkv"], hq, s["q_weight"], s["k_weight"], EPS, s["k_pages"], s["v_pages"], s["table"],
                                              lens, s["row_start"], pos=s["pos"], inv_freq=s["freq"],
                                              interleaved=case["interleaved"], factor=s["factor"],
                                              mrope_section=SECTIONS if case["axes"] == 3 else None, advance=case["first"])
        return q, s["k_pages"], s["v_pages"], lens
    if case["first"]:
        lens += s["row_start"][1:] - s["row_start"][:-1]
    page, place, at = _slots(s)
    pos = at if s["pos"] is None else s["pos"]
    rows = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([hq * d, hkv * d, hkv * d], 1)
    q = _plain_turn(q.view(rows, hq, d), s["q_weight"], pos, s["freq"], s["factor"], case["interleaved"])
    s["k_pages"][page, :, place] = _plain_turn(k.view(rows, hkv, d), s["k_weight"], pos, s["freq"], s["factor"], case["interleaved"])
    s["v_pages"][page, :, place] = v.view(rows, hkv, d)
    return q, s["k_pages"], s["v_pages"], lens


def _run_attend(s):
    case = s["case"]
    if own:
        from axono_b200 import ops

        return ops.gqa_attention_portions_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["row_start"], s["longest"],
                                                window=case["window"])
    hkv, d, page = case["hkv"], case["d"], case["page"]
    group = case["hq"] // hkv
    out = torch.empty_like(s["q"])
    row = 0
    for b, (n, cached) in enumerate(_counts(case)):
        blocks = s["table"][b, :-(-(n + cached) // page)].long()
        k, v = (pool[blocks].transpose(0, 1).reshape(hkv, -1, d)[:, :n + cached].float() for pool in (s["k_pages"], s["v_pages"]))
        keys = torch.arange(n + cached, device=DEV)
        for first in range(0, n, 1024):  # scores of at most 1024 rows at a time
            m = min(1024, n - first)
            at = cached + first + torch.arange(m, device=DEV)
            hidden = keys > at[:, None]
            if case["window"]:
                hidden |= keys <= at[:, None] - case["window"]
            q = s["q"][row + first:row + first + m].float().view(m, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, group * m, d)
            scores = (torch.matmul(q, k.transpose(1, 2)) / math.sqrt(d)).view(hkv, group, m, -1).masked_fill(hidden, -math.inf)
            weights = torch.exp(scores - scores.amax(-1, keepdim=True))
            sums = torch.matmul(weights.view(hkv, group * m, -1), v).view(hkv, group, m, d) / weights.sum(-1, keepdim=True)
            out[row + first:row + first + m] = sums.permute(2, 0, 1, 3).reshape(m, hkv * group, d).to(out.dtype)
        row += n
    return out


def run(state):
    return {"turn": _run_turn, "append": _run_append, "attend": _run_attend}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    e, hq, hkv, d = DTYPES[case["dtype"]].itemsize, case["hq"], case["hkv"], case["d"]
    if case["kind"] == "turn":
        rows = case["rows"]
        return {"bytes": rows * (2 * (hq + hkv) * d * e + 8 * case["axes"]), "flops": rows * (hq + hkv) * d * 8}
    counts = _counts(case)
    rows = sum(n for n, _ in counts)
    if case["kind"] == "append":
        return {"bytes": rows * (2 * (hq + 2 * hkv) * d * e + (24 if case["axes"] == 3 else 0)), "flops": rows * (hq + hkv) * d * 8}
    seen = pairs = 0
    for n, cached in counts:
        w = case["window"] or n + cached
        seen += n + cached - max(0, cached + 1 - w)
        pairs += sum(min(cached + i + 1, w) for i in range(n))
    return {"bytes": 2 * rows * hq * d * e + 2 * seen * hkv * d * e, "flops": 4 * pairs * hq * d}


# ---- the same in 64 bits --------------------------------------------------------------------------------------------------

def _exact_turn(x, weight, pos, freq, factor, interleaved):
    """The rotation as a product of complex numbers."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    pairs = freq.numel()
    head, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
    if pos.dim() == 2:
        pos = torch.stack([pos[axis] for axis in _axis_of_pair(pairs).tolist()], -1)
    else:
        pos = pos[:, None].expand(-1, pairs)
    z = torch.complex(*(head.unflatten(-1, (pairs, 2)).unbind(-1) if interleaved else head.unflatten(-1, (2, pairs)).unbind(-2)))
    z = z * torch.polar(torch.full_like(freq, factor), pos.double() * freq)[:, None, :]
    out = torch.stack([z.real, z.imag], -1 if interleaved else -2).flatten(-2)
    return torch.cat([out, rest], -1)


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    turn = lambda x, w, pos: _exact_turn(x, w, pos, s["freq"], s["factor"], case["interleaved"])  # noqa: E731
    if case["kind"] == "turn":
        return turn(s["q"], s["q_weight"], s["pos"]), turn(s["k"], s["k_weight"], s["pos"])
    counts, page = _counts(case), case["page"]
    if case["kind"] == "append":
        q, k, v = s["qkv"].double().split([hq * d, hkv * d, hkv * d], 1)
        at = torch.cat([torch.arange(cached, cached + n) for n, cached in counts]).to(DEV)
        pos = at if s["pos"] is None else s["pos"]
        q, k, v = turn(q.unflatten(1, (hq, d)), s["q_weight"], pos), turn(k.unflatten(1, (hkv, d)), s["k_weight"], pos), v.unflatten(1, (hkv, d))
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        row = 0
        for b, (n, cached) in enumerate(counts):
            blocks = s["table"][b].long()
            for pool, new in zip(pools, (k, v)):
                flat = pool[blocks].transpose(1, 2).reshape(-1, hkv, d)
                flat[cached:cached + n] = new[row:row + n]
                used = -(-(n + cached) // page)
                pool[blocks[:used]] = flat.unflatten(0, (-1, page)).transpose(1, 2)[:used]
            row += n
        return q, pools[0], pools[1], s["lens"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for b, (n, cached) in enumerate(counts):
        blocks = s["table"][b, :-(-(n + cached) // page)].long()
        for h in range(hq):
            k, v = (pool[blocks, h // (hq // hkv)].reshape(-1, d)[:n + cached].double() for pool in (s["k_pages"], s["v_pages"]))
            for first in range(0, n, 2048):
                m = min(2048, n - first)
                lo = max(0, cached + first + 1 - case["window"]) if case["window"] else 0  # keys before are hidden from all
                logits = s["q"][row + first:row + first + m, h].double() @ k[lo:].T * d ** -0.5
                distance = torch.arange(cached + first, cached + first + m, device=DEV)[:, None] - torch.arange(lo, n + cached, device=DEV)
                seen = (distance >= 0) & ((distance < case["window"]) if case["window"] else True)
                out[row + first:row + first + m, h] = torch.softmax(logits.where(seen, -math.inf), -1) @ v[lo:]
        row += n
    return out
