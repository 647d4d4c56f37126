"""Plain evaluations in 64 bits of the operators for portions, and the caches and tables that their tests run on."""
import math

import torch


def axis_of(i, section):
    _, h, w = section
    return 1 if i % 3 == 1 and i < 3 * h else 2 if i % 3 == 2 and i < 3 * w else 0


def turn(x, weight, eps, pos, inv_freq, interleaved=False, factor=1.0, section=None):
    """x (rows, heads, d) -> norm per head, then the rotation of its first 2 * len(inv_freq) elements; pos (rows) or (3, rows)."""
    y = x.double()
    if weight is not None:
        y = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
    y = y.clone()
    if inv_freq is None:
        return y
    n = inv_freq.numel()
    for i in range(n):
        p = pos if section is None else pos[axis_of(i, section)]
        angle = p.double() * inv_freq[i].double()
        c, s = factor * angle.cos()[:, None], factor * angle.sin()[:, None]
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        a, b = y[..., ia].clone(), y[..., ib].clone()
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def row_table(counts, first=0, device="cuda"):
    starts = [first]
    for n in counts:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device=device)


class Cache:
    """Pools of scattered pages for sequences of `lens` tokens (and room for `more` each), with token-major values beside them."""

    def __init__(self, lens, hkv, d, dtype, page=64, seed=0, poison=math.nan, more=0, scale=1.0, spare=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.page, self.hkv, self.d = page, hkv, d
        blocks = [-(-(n + more) // page) for n in lens]
        total = sum(blocks) + spare
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.full((len(lens), max(max(blocks), 1)), total + 7, dtype=torch.int32)  # outside the pool where unused
        at = 0
        for b, n in enumerate(blocks):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.table = self.table.cuda()
        self.k_pages, self.v_pages = (torch.full((total, hkv, page, d), poison, dtype=dtype, device="cuda") for _ in range(2))
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            pair = [(scale * torch.randn((n, hkv, d), generator=g, device="cuda")).to(dtype) for _ in range(2)]
            self.write(b, 0, *pair)
            self.k.append(pair[0])
            self.v.append(pair[1])
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def place(self, b, start, n):
        at = torch.arange(start, start + n, device="cuda")
        return self.table[b, at // self.page].long(), at % self.page

    def write(self, b, start, k, v):
        page, place = self.place(b, start, k.shape[0])
        self.k_pages[page, :, place], self.v_pages[page, :, place] = k, v

    def read(self, b, start, n):
        page, place = self.place(b, start, n)
        return self.k_pages[page, :, place], self.v_pages[page, :, place]


def attend(q, k, v, start, window=0):
    """Rows q (n, hq, d) at positions start.. over k, v (len, hkv, d): the result, and sum of weight * |value| (which errors of the
    weights scale with; each weight at least 2^-21 of the largest possible, 1, below which an fp16 weight is subnormal and off by 2^-32)
    and the largest |score|."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, mag, top = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0.0
    pos = start + torch.arange(n, device=q.device)[:, None]
    keys = torch.arange(k.shape[0], device=q.device)[None]
    seen = (keys <= pos) & ((keys > pos - window) if window else (keys >= 0))
    for h in range(hq):
        s = (q[:, h].double() @ k[:, h // group].double().T / math.sqrt(d)).masked_fill(~seen, -math.inf)
        some = seen.any(1)
        w = torch.softmax(s[some], -1)
        vh = v[:, h // group].double()
        hidden = (~torch.isfinite(vh)).any(1)
        if hidden.any():  # 0 * inf: the sum over what a row sees
            for i, r in enumerate(some.nonzero()[:, 0].tolist()):
                out[r, h] = w[i][seen[r]] @ vh[seen[r]]
                mag[r, h] = (w[i][seen[r]] + 2.0 ** -21) @ vh[seen[r]].abs()
        else:
            out[some, h], mag[some, h] = w @ vh, (w + 2.0 ** -21 * seen[some]) @ vh.abs()
        if some.any():
            top = max(top, float(s[some][seen[some]].abs().max()))
    return out, mag, top


def attend_all(q, cache, counts, starts, window=0):
    """The same for all rows of a launch; rows of no sequence are left out of the list of (row slice, result, magnitude, top)."""
    out = []
    for b, n in enumerate(counts):
        if n:
            rows = slice(starts[b], starts[b] + n)
            length = int(cache.lens[b])
            out.append((rows, *attend(q[rows], cache.k[b], cache.v[b], length - n, window)))
    return out


def attend_tolerance(dtype, ref, mag, top):
    """The result's rounding; scores in fp32, off by 2^-21 of the largest, and an exponential by 2^-21, which change a weight by as
    much; and in fp16 the weights' own rounding (half a step, 2^-11) before they meet the values.  A result below the smallest normal
    number is rounded to a multiple of that number times eps, so that half of this is added."""
    half = torch.finfo(dtype).eps / 2
    subnormal = torch.finfo(dtype).smallest_normal * half
    weights = 2.0 ** -21 * (2 + 2 * top) + (2.0 ** -11 if dtype == torch.float16 else 0.0)
    return ref.abs() * half * (1 + 2.0 ** -10) + mag * weights + subnormal
