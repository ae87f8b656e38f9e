"""Operators of models that read images, sound or video beside a text, as measurable cases.

Four operators of a serving program's attention layers and of its page manager, each case one call of one of them:

``axes``   norms of the queries and keys of each head and the rotation by positions on several axes (time, height, width);
``cross``  attention of tokens to an encoder's states in a paged cache, one length per user, no causal limit;
``copy``   copies of whole blocks of the paged caches of all layers: forks of sequences, moves of pages;
``keep``   compaction of sequences in the paged caches of all layers: chosen tokens move together, the others are dropped.

Lengths of a batch are spread evenly over the logarithm of [len_lo, len_hi] and shuffled by the seed, so the work of
a case does not depend on the seed.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

# (query heads, KV heads, head size) of the layers: the shapes of the benchmark and of the tests
_HEADS = [(8, 8, 64), (8, 2, 64), (64, 8, 64), (16, 16, 64), (16, 16, 128), (16, 8, 128), (32, 8, 128), (40, 8, 128),
          (64, 8, 128), (16, 8, 256)]
_EPS = 1e-6

# a drawn case costs no more than the largest listed ones
_MAX_BYTES, _MAX_FLOPS = 1.2e9, 2.8e11
_MOST_SCORES = 1 << 30  # of the plain form's attention, which holds all of them


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def _case(kind, heads, **more):
    hq, hkv, d = heads
    return {"kind": kind, "q_heads": hq, "kv_heads": hkv, "head_size": d, **more}


def _axes(tokens, heads, axes, rotary, order="sections", norm=True, interleaved=False):
    """order: each axis a stretch of the pairs ("sections"), or the axes in turn ("alternating")."""
    return _case("axes", heads, tokens=tokens, axes=axes, rotary=rotary, order=order, norm=norm, interleaved=interleaved)


def _cross(users, tokens, heads, block, len_lo, len_hi, empty=0):
    return _case("cross", heads, block=block, users=users, tokens=tokens, len_lo=len_lo, len_hi=len_hi, empty=empty)


def _copy(pairs, layers, heads, block, bits=16):
    return _case("copy", heads, block=block, pairs=pairs, layers=layers, bits=bits)


def _keep(users, layers, heads, block, len_lo, len_hi, share=0.5, drafted=0):
    """Of every sequence's last ``drafted`` tokens (0: of all behind the first quarter) the given share stays."""
    return _case("keep", heads, block=block, users=users, layers=layers, len_lo=len_lo, len_hi=len_hi, share=share, drafted=drafted)


def listed():
    small, l8b, l70b = (8, 8, 64), (32, 8, 128), (64, 8, 128)
    return [
        # one token of each of a few requests: what every layer of a step starts with
        dict(_axes(8, l8b, 3, 128), name="axes-token"),
        # the prompts of a pass, text around frames of a video, views of one projection's output
        dict(_axes(8191, l8b, 3, 128, "alternating"), name="axes-prompt"),
        # the patches of an image in its encoder: rows and columns, no norm
        dict(_axes(4900, (16, 16, 64), 2, 64, norm=False), name="axes-patches"),
        # one token of one request, a short recording
        dict(_cross(1, 1, small, 32, 377, 377), name="cross-token"),
        # a serving batch of an 8B model over images of different sizes; two requests have none
        dict(_cross(32, 1, l8b, 64, 256, 4096, empty=2), name="cross-step"),
        # drafted tokens of a few requests of a 70B model
        dict(_cross(8, 5, l70b, 64, 512, 6404), name="cross-draft"),
        # the beginning of a transcription: texts of odd length over half a minute of sound each
        dict(_cross(4, 447, (16, 16, 64), 32, 1500, 1500), name="cross-text"),
        # prompts of an 8B model over its images
        dict(_cross(2, 2048, l8b, 64, 1601, 6404), name="cross-prompt"),
        # one sequence forked: its last block in every layer
        dict(_copy(1, 32, l8b, 64), name="copy-fork"),
        # the pages of many sequences brought together, 8-bit caches with their scales and bounds
        dict(_copy(250, 12, l8b, 64, bits=8), name="copy-pages"),
        # a verified tree of drafted tokens per request: the accepted path stays
        dict(_keep(32, 32, l8b, 64, 512, 4096, 0.4, drafted=16), name="keep-drafted"),
        # half of an image's tokens dropped behind the first layers' choice
        dict(_keep(4, 16, l8b, 64, 2048, 8192, 0.5), name="keep-half"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["axes", "axes", "cross", "cross", "cross", "copy", "keep"])
        heads, block = rng.choice(_HEADS), rng.choice([32, 64, 128])
        if kind == "axes":
            rotary = rng.choice([heads[2], heads[2], heads[2] // 2])
            case = _axes(_log(rng, 1, 16384), heads, rng.choice([2, 3, 3, 4]), rotary, rng.choice(["sections", "alternating"]),
                         rng.random() < 0.7, rng.random() < 0.3)
        elif kind == "cross":
            users, tokens = _log(rng, 1, 96), rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
            lo = _log(rng, 1, 4096)
            case = _cross(users, tokens, heads, block, lo, min(8192, _log(rng, lo, 16 * lo)), rng.choice([0, 0, users // 6]))
        elif kind == "copy":
            bits = rng.choice([16, 16, 8])  # (a layer has two tensors, or five: 64 of them at most)
            case = _copy(_log(rng, 1, 300), _log(rng, 1, 32 if bits == 16 else 12), heads, block, bits)
        else:
            lo = _log(rng, 64, 4096)
            drafted = rng.choice([0, 0, _log(rng, 4, 64)])
            case = _keep(_log(rng, 1, 48), _log(rng, 1, 32), heads, block, lo, min(16384, _log(rng, lo, 8 * lo)),
                         rng.choice([0.1, 0.5, 0.9]), drafted)
        w = work(case)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS and _held_bytes(case) <= 4e9 and _scores(case) <= _MOST_SCORES:
            return case


# --------------------------------------------------------------------------- #
# sizes
# --------------------------------------------------------------------------- #
def _lengths(case):
    """One entry per user that has any."""
    n = case["users"] - case.get("empty", 0)
    lo, hi = case["len_lo"], case["len_hi"]
    return [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]


def _first_and_kept(case, length):
    """The first position that a sequence's compaction touches, and how many tokens stay from there on."""
    first = max(length - case["drafted"], 0) if case["drafted"] else length // 4
    return first, max(1, int((length - first) * case["share"]))


def _block_bytes(case):
    """Of all tensors of a layer."""
    hkv, bs, d = case["kv_heads"], case["block"], case["head_size"]
    if case["bits"] == 16:
        return 2 * hkv * bs * d * 2
    return 2 * hkv * bs * d + 2 * hkv * 4 + hkv * 2 * d * 2


def _held_bytes(case):
    if case["kind"] == "copy":
        return 2 * case["pairs"] * case["layers"] * _block_bytes(case)
    if case["kind"] == "keep":
        rows = sum((n - 1) // case["block"] - _first_and_kept(case, n)[0] // case["block"] + 1 for n in _lengths(case)) * case["block"]
        return rows * case["layers"] * 4 * case["kv_heads"] * case["head_size"]
    if case["kind"] == "cross":
        return sum(_lengths(case)) * 4 * case["kv_heads"] * case["head_size"]
    return 0


def _scores(case):
    return case["users"] * case["q_heads"] * case["tokens"] * case["len_hi"] if case["kind"] == "cross" else 0


def work(case):
    hq, hkv, d, kind = (case[k] for k in ("q_heads", "kv_heads", "head_size", "kind"))
    if kind == "axes":
        n = case["tokens"]
        # rows read and written, a position per axis, and each row of the table that a token may be the first to name
        return {"bytes": n * ((hq + hkv) * d * 4 + case["axes"] * 4 + case["rotary"] * 4), "flops": n * (hq + hkv) * d * 7.0}
    if kind == "cross":
        seen = _lengths(case)
        return {"bytes": sum(seen) * 4 * hkv * d + sum(-(-n // case["block"]) for n in seen) * 4 + case["users"] * case["tokens"] * hq * d * 4,
                "flops": 4.0 * d * hq * case["tokens"] * sum(seen)}
    if kind == "copy":
        return {"bytes": case["pairs"] * (2 * case["layers"] * _block_bytes(case) + 8), "flops": 0.0}
    rows = sum(_first_and_kept(case, n)[1] for n in _lengths(case))
    return {"bytes": rows * (case["layers"] * 2 * hkv * d * 2 * 2 + 4), "flops": 0.0}


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _filled(gen, *shape):
    """Large caches: a stretch of random numbers, repeated."""
    out = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
    flat = out.view(-1)
    some = _randn(gen, min(flat.numel(), (1 << 22) + 4099))
    for at in range(0, flat.numel(), some.numel()):
        flat[at : at + some.numel()] = some[: flat.numel() - at]
    return out


def _table(host, need, width):
    """Block tables of users that hold ``need`` blocks each, out of one shuffled pool; -1 where a user has none."""
    total = sum(need)
    order = host.permutation(total)
    table = np.full((len(need), width), -1, dtype=np.int32)
    at = 0
    for u, n in enumerate(need):
        table[u, :n] = order[at : at + n]
        at += n
    return max(total, 1), table


def _grid_positions(host, tokens, axes):
    """[axes, tokens]: a stretch of text (the same number on all axes), frames of rows and columns, and text again, which goes
    on behind the largest number so far."""
    if axes == 2:  # an image in its encoder: rows and columns alone
        side = max(1, int(math.isqrt(tokens)))
        at = np.arange(tokens)
        return np.stack([at // side, at % side]).astype(np.int32)
    start = int(host.integers(0, 512)) if tokens < 64 else 0
    text = max(1, tokens // 8)
    grid = max(0, tokens - 2 * text)
    side = max(1, int(math.isqrt(max(1, grid // 8))))
    at = np.arange(grid)
    numbers = [at // (side * side), at // side % side, at % side, at % 2][:axes]
    first = np.tile(start + np.arange(text), (axes, 1))
    middle = np.stack(numbers) + start + text
    top = (int(middle.max()) if grid else start + text - 1) + 1
    last = np.tile(top + np.arange(tokens - text - grid), (axes, 1))
    return np.concatenate([first, middle, last], 1).astype(np.int32)[:, :tokens]


def _pair_axes(case):
    """The axis of every pair of features."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    if case["order"] == "alternating":
        return np.arange(pairs) % axes
    # the first axis a quarter, the others share the rest evenly; two axes half each
    first = pairs // 2 if axes == 2 else pairs // 4
    rest = np.arange(pairs - first) * (axes - 1) // (pairs - first) + 1
    return np.concatenate([np.zeros(first, dtype=np.int64), rest])


def _angles(positions, rotary):
    """The program's table of cosines and sines, [positions, rotary], computed once."""
    f = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] \
        * 500000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    return torch.cat([f.cos(), f.sin()], 1).float()


def prepare(case, seed):
    if "tt-xla_amd" not in "".join(sys.path):
        sys.path.insert(0, os.path.abspath("tt-xla_amd"))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    hq, hkv, d, kind = (case[k] for k in ("q_heads", "kv_heads", "head_size", "kind"))
    s = {"kind": kind, "case": dict(case)}
    if kind == "axes":
        n = case["tokens"]
        qkv = _randn(gen, n, (hq + 2 * hkv) * d)  # queries, keys and values of one projection
        s["q"], s["k"], _ = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
        s["weights"] = tuple(1 + 0.2 * _randn(gen, d) for _ in range(2)) if case["norm"] else (None, None)
        positions = _grid_positions(host, n, case["axes"])
        s["positions"] = torch.from_numpy(positions).cuda()
        s["pair_axes"] = torch.from_numpy(_pair_axes(case).astype(np.int32)).cuda()
        s["angles"] = _angles(int(positions.max()) + 1, case["rotary"])
        return s
    bs = case["block"]
    if kind == "cross":
        users = case["users"]
        lens = np.zeros(users, dtype=np.int64)
        lens[: users - case["empty"]] = _lengths(case)
        lens = host.permutation(lens)
        blocks, table = _table(host, [-(-int(n) // bs) for n in lens], -(-case["len_hi"] // bs))
        s["table"], s["lens"] = torch.from_numpy(table).cuda(), torch.from_numpy(lens.astype(np.int32)).cuda()
        s["cache"] = tuple(_filled(gen, blocks, hkv, bs, d) for _ in range(2))
        q = _randn(gen, users * case["tokens"], hq * d)
        s["q"] = q.view(users, case["tokens"], hq, d).transpose(1, 2)
        s["most"] = int(lens.max())
        return s
    if kind == "copy":
        pairs = case["pairs"]
        order = host.permutation(2 * pairs).astype(np.int32)
        s["source"], s["target"] = (torch.from_numpy(x.copy()).cuda() for x in (order[:pairs], order[pairs:]))
        s["caches"] = []
        for _ in range(case["layers"]):
            kv = [_filled(gen, 2 * pairs, hkv, bs, d) for _ in range(2)]
            if case["bits"] == 8:
                bounds = torch.stack([kv[0].amin(2), kv[0].amax(2)], 2)
                scales = [torch.ldexp(torch.ones(2 * pairs, hkv, device="cuda"), torch.randint(-9, -6, (2 * pairs, hkv), generator=gen, device="cuda"))
                          for _ in range(2)]
                kv = [x.to(torch.float8_e4m3fn) for x in kv] + scales + [bounds]
            s["caches"] += kv
        return s
    lens = host.permutation(np.array(_lengths(case), dtype=np.int64))
    plan = [_first_and_kept(case, int(n)) for n in lens]
    # the blocks in front of a sequence's first touched position are one block that nothing reads or writes
    skip, width = [f // bs for f, _ in plan], -(-int(lens.max()) // bs)
    blocks, touched = _table(host, [-(-int(n) // bs) - m for n, m in zip(lens, skip)], width)
    table = np.full_like(touched, blocks)
    for u, m in enumerate(skip):
        table[u, m:] = touched[u, : width - m]
    kept = np.zeros((len(lens), max(k for _, k in plan)), dtype=np.int32)
    for u, (first, n) in enumerate(plan):
        kept[u, :n] = first + np.sort(host.permutation(int(lens[u]) - first)[:n])
    s["table"], s["kept"] = torch.from_numpy(table).cuda(), torch.from_numpy(kept).cuda()
    s["first"] = torch.tensor([f for f, _ in plan], dtype=torch.int32, device="cuda")
    s["kept_lens"] = torch.tensor([n for _, n in plan], dtype=torch.int32, device="cuda")
    s["caches"] = [_filled(gen, blocks + 1, hkv, bs, d) for _ in range(2 * case["layers"])]
    return s


# --------------------------------------------------------------------------- #
# the plain forms
# --------------------------------------------------------------------------- #
def _turned(x, weight, cos, sin, interleaved):
    """RMS norm and rotation of rows [tokens, heads, head size] in float32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    half = cos.shape[-1]
    turn, rest = x[..., : 2 * half], x[..., 2 * half :]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turn[..., :half], turn[..., half:]
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turn, rest], -1).to(torch.bfloat16)


def _plain_axes(s):
    # a pair's row of the table is named by the position on its axis
    rows = s["positions"].long()[s["pair_axes"].long()].t()  # [tokens, pairs]
    at = torch.arange(rows.shape[1], device="cuda")
    cos, sin = (s["angles"][rows, at + shift][:, None, :] for shift in (0, rows.shape[1]))
    turned = s["case"]["interleaved"]
    return _turned(s["q"], s["weights"][0], cos, sin, turned), _turned(s["k"], s["weights"][1], cos, sin, turned)


def _plain_cross(s):
    c = s["case"]
    b, hq, n, d = s["q"].shape
    hkv = c["kv_heads"]
    table = s["table"].clamp(min=0).long()
    k, v = (x[table].transpose(1, 2).flatten(2, 3).float() for x in s["cache"])  # [users, kv heads, keys, d]
    q = s["q"].float().reshape(b, hkv, -1, d)
    w = (q @ k.transpose(2, 3)) * d**-0.5
    masked = (torch.arange(k.shape[2], device="cuda")[None, :] >= s["lens"][:, None])[:, None, None, :]
    w = w.masked_fill(masked, -torch.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    out = (w @ v) / torch.where(total == 0, torch.ones_like(total), total)  # nothing to attend: zeros
    return out.view(b, hq, n, d).to(torch.bfloat16)


def _bytes(x):
    return x.view(torch.uint8) if x.dtype.itemsize == 1 else x


def _plain_copy(s):
    for cache in s["caches"]:
        x = _bytes(cache)
        x[s["target"].long()] = x[s["source"].long()]
    return s["caches"]


def _plain_keep(s):
    bs, users, most = s["case"]["block"], s["kept"].shape[0], s["kept"].shape[1]
    at = torch.arange(most, device="cuda")
    user = torch.arange(users, device="cuda")[:, None].expand(-1, most)
    live = at[None, :] < s["kept_lens"][:, None]
    source, target = s["kept"].long()[live], (s["first"].long()[:, None] + at)[live]
    table, user = s["table"].long(), user[live]
    for cache in s["caches"]:
        rows = cache[table[user, source // bs], :, source % bs]
        cache[table[user, target // bs], :, target % bs] = rows
    return s["caches"]


# --------------------------------------------------------------------------- #
# the framework's calls
# --------------------------------------------------------------------------- #
def _own(s):
    import tt_xla_amd  # noqa: F401  (registers the operators)

    tt, kind = torch.ops.tt, s["kind"]
    if kind == "axes":
        return tt.qk_norm_rope_axes(s["q"], s["k"], s["angles"], s["positions"], s["pair_axes"], *s["weights"], _EPS,
                                    s["case"]["interleaved"])
    if kind == "cross":
        return tt.paged_cross_attention(s["q"], *s["cache"], s["table"], s["lens"], most_keys=s["most"])
    if kind == "copy":
        tt.copy_cache_blocks_(s["caches"], s["source"], s["target"])
    else:
        tt.keep_cache_tokens_(s["caches"], s["table"], s["kept"], s["kept_lens"], s["first"])
    return s["caches"]


_PLAIN = {"axes": _plain_axes, "cross": _plain_cross, "copy": _plain_copy, "keep": _plain_keep}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["kind"]](state)


# --------------------------------------------------------------------------- #
# the definitions in 64 bits
# --------------------------------------------------------------------------- #
def _exact_rows(x, weight, spin, interleaved):
    """[tokens, heads, d] float64: every pair of features turned as a complex number."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * weight.double()
    half = spin.shape[1]
    out = x.clone()
    at = torch.arange(half, device=x.device)
    one, two = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * spin[:, None, :]
    out[..., one], out[..., two] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, kind = case["q_heads"], case["kv_heads"], case["kind"]
    if kind == "axes":
        pairs = case["rotary"] // 2
        spin = torch.empty(case["tokens"], pairs, dtype=torch.complex128, device="cuda")
        for j, axis in enumerate(s["pair_axes"].tolist()):
            row = s["angles"].double()[s["positions"][axis].long()]
            spin[:, j] = torch.complex(row[:, j].contiguous(), row[:, pairs + j].contiguous())
        return [_exact_rows(s[t], s["weights"][i], spin, case["interleaved"]) for i, t in enumerate("qk")]
    if kind == "cross":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        g, bs, d = hq // hkv, case["block"], case["head_size"]
        for u, n in enumerate(s["lens"].tolist()):
            pages = s["table"][u, : -(-n // bs)].long()
            for h in range(hkv if n else 0):
                k, v = (x[pages, h].flatten(0, 1)[:n].double() for x in s["cache"])
                w = s["q"][u, h * g : h * g + g].double().reshape(-1, d) @ k.t().contiguous() / math.sqrt(d)
                out[u, h * g : h * g + g] = (torch.softmax(w, -1) @ v).view(g, -1, d)
        return out
    if kind == "copy":
        for source, target in zip(s["source"].tolist(), s["target"].tolist()):
            for cache in s["caches"]:
                _bytes(cache)[target].copy_(_bytes(cache)[source])
        return s["caches"]
    bs = case["block"]
    for u, (first, n) in enumerate(zip(s["first"].tolist(), s["kept_lens"].tolist())):
        pages = s["table"][u].long()
        pages = pages[pages >= 0]
        for cache in s["caches"]:
            rows = cache[pages].transpose(1, 2).flatten(0, 1)  # [positions, heads, d]
            rows[first : first + n] = rows[s["kept"][u, :n].long()]
            cache[pages] = rows.unflatten(0, (-1, bs)).transpose(1, 2)
    return s["caches"]
