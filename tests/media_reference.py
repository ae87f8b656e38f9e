"""Rotation by several axes, cross attention, block copies and compaction, plainly and in 64 bits, for their tests (CPU tensors)."""

import torch

import fp8_reference as R


def turn_axes(x, weight, table, positions, pair_axes, eps, interleaved):
    """Norm and rotation of x [tokens, heads, d] in float64, pair j by the position [axes, tokens] on axis pair_axes[j]; a pair whose axis does
    not exist or whose position is outside the table is not turned."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    half = table.shape[1] // 2
    out = x.clone()
    for j, axis in enumerate(pair_axes.tolist()):
        if not 0 <= axis < positions.shape[0]:
            continue
        pos = positions[axis]
        known = (pos >= 0) & (pos < table.shape[0])
        row = table.double()[pos.clamp(0, table.shape[0] - 1).long()]
        cos = torch.where(known, row[:, j], torch.ones(()).double())[:, None]
        sin = torch.where(known, row[:, half + j], torch.zeros(()).double())[:, None]
        p, q = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        out[..., p] = x[..., p] * cos - x[..., q] * sin
        out[..., q] = x[..., q] * cos + x[..., p] * sin
    return out


def cross(q, k_cache, v_cache, table, lens, scale, room=None):
    """q [users, heads, tokens, d] -> (out, spread) float64: softmax over the first lens[u] keys of every user, zeros over none; spread = sum p |v|."""
    users, hq, s, d = q.shape
    nb, hkv, bs, _ = k_cache.shape
    out, spread = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    g = hq // hkv
    for u in range(users):
        n = min(int(lens[u]), table.shape[1] * bs if room is None else room)
        if n <= 0:
            continue
        ids = [i if 0 <= i < nb else 0 for i in table[u, : -(-n // bs)].tolist()]
        for h in range(hkv):
            k, v = (c[ids, h].flatten(0, 1)[:n].double() for c in (k_cache, v_cache))
            rows = q[u, h * g : h * g + g].reshape(-1, d)
            o, w = R.softmax_rows(rows, k, v, torch.ones(rows.shape[0], n, dtype=torch.bool), scale)
            out[u, h * g : h * g + g], spread[u, h * g : h * g + g] = o.view(g, s, d), w.view(g, s, d)
    return out, spread


def copy_blocks(caches, source, target):
    """As if the pairs went one after the other."""
    for s, t in zip(source.tolist(), target.tolist()):
        for c in caches:
            if 0 <= s < c.shape[0] and 0 <= t < c.shape[0]:
                c[t] = c[s].clone()


def keep_tokens(cache, table, kept, kept_lens, first=None):
    """What a cache [num_blocks, heads, block, d] holds afterwards."""
    nb, _, bs, _ = cache.shape
    out, room = cache.clone(), table.shape[1] * bs
    for u in range(table.shape[0]):
        start = 0 if first is None else int(first[u])
        for i in range(max(0, min(int(kept_lens[u]), kept.shape[1]))):
            s, d = int(kept[u, i]), start + i
            if not (0 <= d <= s < room):
                continue
            ps, pd = int(table[u, s // bs]), int(table[u, d // bs])
            if 0 <= ps < nb and 0 <= pd < nb:
                out[pd, :, d % bs] = cache[ps, :, s % bs]
    return out
