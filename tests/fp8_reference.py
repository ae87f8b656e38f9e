"""The operators around the 8-bit cache, plainly and in 64 bits, for their tests (CPU tensors)."""

import math

import torch

MAX = 448.0
LEAST, MOST = -110, 119  # exponents of a scale


def nearest_e4m3(x):
    """float64 -> nearest e4m3 value, ties to even; beyond the range the largest, infinities NaN."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    y = (torch.round(x / step) * step).clamp(-MAX, MAX)
    return torch.where(torch.isfinite(x), y, torch.full_like(x, math.nan))


def scale_for(x):
    """The scale of values x [..., rows, d]: [...]."""
    most = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).flatten(-2).amax(-1)
    s = torch.full_like(most, 2.0**LEAST)
    for e in range(LEAST + 1, MOST + 1):
        s = torch.where(most > MAX * 2.0 ** (e - 1), torch.full_like(s, 2.0**e), s)
    return s


def values(elements):
    """e4m3 elements -> float64."""
    return elements.to(torch.float32).to(torch.float64)


class Cache:
    """K and V caches, scales and bounds as float64 tensors, written as the operators are documented to write them."""

    def __init__(self, k, v, ks, vs, bounds=None):
        self.e = [values(k.cpu()), values(v.cpu())]
        self.s = [ks.cpu().double(), vs.cpu().double()]
        self.b = None if bounds is None else bounds.cpu().double()

    def _rows(self, i, block, row, x):
        """x [hkv, n, d] to rows row .. row + n - 1 of a block."""
        e, s = self.e[i], self.s[i]
        old = s[block] if row else torch.zeros_like(s[block])
        new = torch.maximum(old, scale_for(x))
        if row:
            e[block, :, :row] = nearest_e4m3(e[block, :, :row] * (old / new)[:, None, None])
        e[block, :, row : row + x.shape[1]] = nearest_e4m3(x / new[:, None, None])
        s[block] = new
        if i == 0 and self.b is not None:
            seen = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x).amin(1), torch.where(
                torch.isnan(x), torch.full_like(x, -math.inf), x).amax(1)
            if row:
                seen = torch.minimum(self.b[block, :, 0], seen[0]), torch.maximum(self.b[block, :, 1], seen[1])
            self.b[block, :, 0], self.b[block, :, 1] = seen

    def update(self, k, v, positions, table):
        """k, v [users, hkv, d]"""
        nb, _, bs, _ = self.e[0].shape
        for u, p in enumerate(positions.tolist()):
            if p < 0 or p // bs >= table.shape[1] or not 0 <= int(table[u, p // bs]) < nb:
                continue
            for i, x in enumerate((k, v)):
                self._rows(i, int(table[u, p // bs]), p % bs, x[u].cpu().double()[:, None])

    def fill(self, k, v, table, rows):
        """k, v [users, hkv, tokens, d]"""
        nb, _, bs, _ = self.e[0].shape
        for n, r in enumerate(rows):
            if not 0 <= r < table.shape[0]:
                continue
            for c in range(-(-k.shape[2] // bs)):
                if 0 <= int(table[r, c]) < nb:
                    for i, x in enumerate((k, v)):
                        self._rows(i, int(table[r, c]), 0, x[n, :, c * bs : c * bs + bs].cpu().double())

    def differences(self, k, v, ks, vs, bounds=None):
        """Where the device's tensors differ (NaN equals NaN)."""
        def differ(a, b):
            return int(((a != b) & ~(torch.isnan(a) & torch.isnan(b))).sum())

        got = {"k": differ(values(k.cpu()), self.e[0]), "v": differ(values(v.cpu()), self.e[1]),
               "k_scales": differ(ks.cpu().double(), self.s[0]), "v_scales": differ(vs.cpu().double(), self.s[1])}
        if bounds is not None:
            got["bounds"] = differ(bounds.cpu().double(), self.b)
        return {n: c for n, c in got.items() if c}


def turn(x, weight, table, positions, eps, interleaved):
    """Norm and rotation of x [tokens, heads, d] in float64; a position outside the table is not turned."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    half = table.shape[1] // 2
    known = (positions >= 0) & (positions < table.shape[0])
    a = table.double()[positions.clamp(0, table.shape[0] - 1).long()]
    cos = torch.where(known[:, None], a[:, :half], torch.ones(()).double())[:, None, :]
    sin = torch.where(known[:, None], a[:, half:], torch.zeros(()).double())[:, None, :]
    out = x.clone()
    i = torch.arange(half)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out[..., p] = x[..., p] * cos - x[..., q] * sin
    out[..., q] = x[..., q] * cos + x[..., p] * sin
    return out


def gather(elements, scales, ids, h):
    """[keys, d] float64 of head h through block ids; ids out of range read block 0."""
    nb = elements.shape[0]
    ids = [i if 0 <= i < nb else 0 for i in ids]
    e = values(elements[ids, h].cpu())
    return (e * scales[ids, h].cpu().double()[:, None, None]).flatten(0, 1)


def softmax_rows(q, k, v, allowed, scale, sink=None):
    """q [n, d], k / v [keys, d], allowed [n, keys] -> (out [n, d], spread [n, d] = sum p |v|)."""
    n = q.shape[0]
    w = (q.double() @ k.T) * scale
    w = torch.where(allowed, w, torch.full_like(w, -math.inf))
    top = w.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.double().reshape(-1, 1).expand(n, 1))
    w = torch.exp(w - top)
    total = w.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink.double().reshape(-1, 1) - top)
    p = w / total
    # an unattended row of V has no part in the result, whatever stands there
    used = allowed.any(0)
    v = torch.where(used[:, None], v, torch.zeros_like(v))
    return p @ v, p @ v.abs()


def block_scores(q, low, high):
    """q [g, d], low / high [blocks, d] -> [blocks]"""
    q, low, high = q.double(), low.double(), high.double()
    s = (q.clamp(min=0)[:, None] * high[None] + q.clamp(max=0)[:, None] * low[None]).sum(-1)
    return torch.where(torch.isfinite(s) | (s == -math.inf), s, torch.full_like(s, math.inf)).amax(0)


def choose(q, bounds, ids, h, blocks, kept):
    """Columns that the sparse decode keeps of a context of `blocks` blocks."""
    if blocks <= kept:
        return list(range(blocks))
    nb = bounds.shape[0]
    ids = [i if 0 <= i < nb else 0 for i in ids[:blocks]]
    s = block_scores(q, bounds[ids, h, 0].cpu(), bounds[ids, h, 1].cpu()).tolist()
    best = sorted(range(1, blocks - 1), key=lambda c: (-s[c], c))[: kept - 2]
    return sorted([0, blocks - 1, *best])
