"""Workloads of the token operators that read the feature maps of the DCNv2 layers: the norm and
position rotation of queries and keys (dcnv2_qk_norm_rotary) and the attention of queries to an
encoder's states (dcnv2_cross_attention).

`run` computes them in their plain form (elementary torch operations in fp32, angles in fp64), or,
with `own` set, through the package's entry points. `exact` is each operator's definition in fp64.

Sizes: 5456 tokens are the five levels 64, 32, 16, 8, 4 of the 512 x 512 detector step (one token
per pixel), 4096 and 16384 tokens the 64 x 64 and 128 x 128 maps, 256 channels are 8 heads of 32.
The other sizes are generic (heads of 64 to 128, single tokens, odd lengths).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LEVELS = (64, 32, 16, 8, 4)
BASE = 10000.0


def _rotary(name, batch, tokens, q_heads, k_heads, dim, dtype, norm, grid, rot=None, order="blocks",
            interleaved=False, shared=False):
    return {"name": name, "op": "rotary", "batch": batch, "tokens": tokens, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "dtype": dtype, "norm": norm, "grid": grid,
            "rot": dim if rot is None else rot, "order": order, "interleaved": interleaved,
            "shared": shared}


def _attention(name, batch, q_tokens, kv_tokens, q_heads, kv_heads, dim, dtype, layout, mask):
    return {"name": name, "op": "attention", "batch": batch, "q_tokens": q_tokens,
            "kv_tokens": kv_tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "layout": layout, "mask": mask}


def listed():
    return [
        # one new token of four sequences in a decoder with grouped heads: launch latency
        _rotary("rot_step", 4, 1, 32, 8, 128, "bf16", True, "line"),
        # fp32 activations of an odd-sized image map, rotated in half of each head only
        _rotary("rot_map_fp32", 3, 1021, 12, 12, 64, "fp32", True, "map", rot=32, shared=True),
        # frames of a video, three axes over the head in turn, neighbouring elements as pairs
        _rotary("rot_video", 2, 7161, 16, 16, 80, "bf16", False, "video", order="turns",
                interleaved=True),
        # keys of the detector step's five levels, batch 32, 256 channels
        _rotary("rot_levels_keys", 32, 5456, 0, 8, 32, "fp16", True, "levels", shared=True),
        # queries and keys of 128 x 128 maps in a wide layer with grouped heads
        _rotary("rot_map_wide", 4, 16384, 32, 8, 128, "bf16", True, "map"),
        # one token of one sequence reads the levels of one image: latency, few rows, one long axis
        _attention("attn_step", 1, 1, 5456, 32, 8, 128, "bf16", "cache", "none"),
        # one token of 32 sequences reads padded images (a rectangle of each level is valid)
        _attention("attn_step_padded", 32, 1, 5456, 8, 8, 32, "fp16", "fused", "pixels"),
        # single tokens over a long cache, lengths from none to all of it
        _attention("attn_step_long", 8, 1, 60001, 64, 8, 128, "bf16", "cache", "lens"),
        # odd sizes everywhere: three sequences, the shortest without any state
        _attention("attn_odd", 3, 197, 1021, 6, 2, 72, "fp16", "fused", "lens"),
        # object queries of a detection decoder over the levels of a padded batch
        _attention("attn_queries", 32, 300, 5456, 8, 8, 32, "fp16", "fused", "pixels"),
        # pixels of 64 x 64 maps read a short text of its own length per image
        _attention("attn_text", 8, 4096, 77, 8, 8, 64, "bf16", "fused", "lens"),
        # pixels of a 64 x 64 map read the states of a 128 x 128 map
        _attention("attn_maps", 1, 4096, 16384, 16, 16, 128, "bf16", "plain", "none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rotary(rng):
    grid = rng.choice(["line", "map", "video", "levels"])
    dim = rng.choice([16, 32, 40, 64, 72, 80, 96, 128, 256])
    axes = {"line": 1, "map": 2}.get(grid, 3)
    rot = rng.choice([dim, dim, dim // 2 // 4 * 4])
    k_heads = rng.choice([0, 1, 2, 4, 8, 12])
    return {"op": "rotary", "batch": _log(rng, 1, 32), "tokens": _log(rng, 1, 17000),
            "q_heads": max(1, k_heads) * rng.choice([1, 1, 2, 4]), "k_heads": k_heads, "dim": dim,
            "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"]), "norm": rng.random() < 0.7,
            "grid": grid, "rot": max(2 * axes, rot),
            "order": rng.choice(["blocks", "blocks", "turns"]),
            "interleaved": rng.random() < 0.3, "shared": rng.random() < 0.5}


def _draw_attention(rng):
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    return {"op": "attention", "batch": _log(rng, 1, 32),
            "q_tokens": 1 if rng.random() < 0.4 else _log(rng, 1, 4200),
            "kv_tokens": _log(rng, 1, 61000), "q_heads": kv_heads * rng.choice([1, 1, 2, 4, 8]),
            "kv_heads": kv_heads, "dim": rng.choice([16, 32, 40, 64, 72, 80, 96, 128]),
            "dtype": rng.choice(["fp16", "bf16"]),
            "layout": rng.choice(["plain", "fused", "cache"]),
            "mask": rng.choice(["none", "lens", "pixels"])}


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most.setdefault(c["op"], []).append((w["bytes"], w["flops"], _scores(c)))
    op = rng.choice(["rotary", "attention"])
    while True:
        case = _draw_rotary(rng) if op == "rotary" else _draw_attention(rng)
        w, top = work(case), most[op]
        if (w["bytes"] <= max(t[0] for t in top) and w["flops"] <= max(t[1] for t in top)
                and _scores(case) <= max(t[2] for t in top)):
            return case


def _scores(case):
    if case["op"] != "attention":
        return 0
    return case["batch"] * case["q_heads"] * case["q_tokens"] * case["kv_tokens"]


# ---------------------------------------------------------------- inputs


def _axes(grid):
    return {"line": 1, "map": 2}.get(grid, 3)


def _pair_axis(case):
    """Axis of each rotated pair: in blocks (the axes one after another) or in turns."""
    n, axes = case["rot"] // 2, _axes(case["grid"])
    if case["order"] == "turns":
        return bytes(i % axes for i in range(n))
    return bytes(min(i * axes // n, axes - 1) for i in range(n))


def _positions(case, g, dev):
    """int32 [batch or 1, tokens, axes]: the grid's coordinates, moved by the text ahead of it."""
    T, n = case["tokens"], 1 if case["shared"] else case["batch"]
    i = torch.arange(T, device=dev)
    if case["grid"] == "line":
        p = i[:, None]
    elif case["grid"] == "map":
        w = max(1, math.isqrt(T))
        p = torch.stack([i // w, i % w], 1)
    elif case["grid"] == "video":
        h = w = max(1, round((T / 7) ** 0.5))
        p = torch.stack([i // (h * w), i // w % h, i % w], 1)
    else:
        sides = torch.tensor(LEVELS, device=dev)
        ends = torch.cumsum(sides * sides, 0)
        j = i % int(ends[-1])
        level = torch.searchsorted(ends, j, right=True)
        j = j - (ends - sides * sides)[level]
        p = torch.stack([level, j // sides[level], j % sides[level]], 1)
    start = torch.randint(0, 100000 if case["grid"] == "line" else 3000, (n, 1, 1), generator=g,
                          device=dev)
    return (p[None] + start).to(torch.int32).contiguous()


def _lengths(case):
    """Lengths of the batch's states, from all of them down; the last of several is empty."""
    B, S = case["batch"], case["kv_tokens"]
    return [S - (S * 3 // 4) * b // max(1, B - 1) if b < B - 1 or B == 1 else 0 for b in range(B)]


def _rects(case):
    """Valid share (height, width) of each image of a padded batch."""
    B = case["batch"]
    return [(1.0 - 0.4 * (b % 5) / 4, 1.0 - 0.5 * (b % 3) / 2) for b in range(B)]


def _sides(S):
    """The maps that S tokens come from: the five levels, or one map about square."""
    if S == sum(s * s for s in LEVELS):
        return LEVELS
    return (max(1, math.isqrt(S)),)


def _valid_pixels(S, rect, dev="cpu"):
    parts, left = [], S
    for k, s in enumerate(_sides(S)):
        i = torch.arange(s * s if len(_sides(S)) > 1 else left, device=dev)
        rows = (len(i) + s - 1) // s
        parts.append((i // s < max(1, math.ceil(rows * rect[0])))
                     & (i % s < max(1, math.ceil(s * rect[1]))))
    return torch.cat(parts)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, B, D = DTYPES[case["dtype"]], case["batch"], case["dim"]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.float32) * std).to(dt)

    if case["op"] == "rotary":
        T, hq, hk = case["tokens"], case["q_heads"], case["k_heads"]
        x = normal(B, T, hq + hk, D, std=1.5)  # one projection gives queries and keys
        n, axes, of = case["rot"] // 2, _axes(case["grid"]), _pair_axis(case)
        if case["order"] == "turns":  # one table over the whole head
            f = [BASE ** (-i / n) for i in range(n)]
        else:  # each axis has a table of its own
            f = [BASE ** (-of[:i].count(a) / of.count(a)) for i, a in enumerate(of)]
        s = {"case": case, "q": x[:, :, :hq] if hq else None, "k": x[:, :, hq:] if hk else None,
             "positions": _positions(case, g, dev), "pair_axis": of,
             "freqs": torch.tensor(f, dtype=torch.float32, device=dev),
             "axis": torch.tensor(list(of), device=dev)}
        s["q_weight"] = (1 + 0.2 * normal(D)).to(dt) if case["norm"] and hq else None
        s["k_weight"] = (1 + 0.2 * normal(D)).to(dt) if case["norm"] and hk else None
        return s
    L, S, hq, hk = case["q_tokens"], case["kv_tokens"], case["q_heads"], case["kv_heads"]
    q = normal(B, L, hq, D)
    if case["layout"] == "fused":  # one projection gives keys and values
        kv = normal(B, S, 2, hk, D)
        k, v = kv[:, :, 0], kv[:, :, 1]
    elif case["layout"] == "cache":  # heads ahead of tokens
        k, v = (normal(B, hk, S, D).transpose(1, 2) for _ in range(2))
    else:
        k, v = (normal(B, S, hk, D) for _ in range(2))
    s = {"case": case, "q": q, "k": k, "v": v, "kv_lens": None, "key_mask": None}
    order = torch.randperm(B, generator=g, device=dev)
    if case["mask"] == "lens":
        s["kv_lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order]
    elif case["mask"] == "pixels":
        kinds = {r: _valid_pixels(S, r, dev) for r in sorted(set(_rects(case)))}
        s["key_mask"] = torch.stack([kinds[r] for r in _rects(case)])[order]
    return s


# ---------------------------------------------------------------- the operators


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "tensorrt-dcnv2-plugin_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dcnv2_b200
    return dcnv2_b200


def _run_own(s):
    dcn = _package()
    if s["case"]["op"] == "rotary":
        q, k = dcn.dcnv2_qk_norm_rotary(
            s["q"], s["k"], s["positions"], s["freqs"], s["pair_axis"], q_weight=s["q_weight"],
            k_weight=s["k_weight"], norm="rms" if s["case"]["norm"] else None, eps=1e-6,
            interleaved=s["case"]["interleaved"])
        return {n: t for n, t in (("q", q), ("k", k)) if t is not None}
    out, lse = dcn.dcnv2_cross_attention(s["q"], s["k"], s["v"], kv_lens=s["kv_lens"],
                                         key_mask=s["key_mask"], return_lse=True)
    return {"out": out, "lse": lse}


def _norm_rotate(x, weight, cos, sin, case):
    y = x.float()
    if case["norm"]:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    rot = case["rot"]
    part, rest = y[..., :rot], y[..., rot:]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([part, rest], -1).to(x.dtype)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "rotary":
        angle = s["positions"][..., s["axis"]].double() * s["freqs"].double()
        cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
        return {n: _norm_rotate(s[n], s[n + "_weight"], cos, sin, case) for n in ("q", "k")
                if s[n] is not None}
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, L, H, D = q.shape
    S, G = k.shape[1], k.shape[2]
    q = q.view(B, L, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * L, D)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(D))  # [B, G, rows, S]
    if s["kv_lens"] is not None:
        gone = torch.arange(S, device=q.device) >= s["kv_lens"][:, None]
        score.masked_fill_(gone[:, None, None], -math.inf)
    if s["key_mask"] is not None:
        score.masked_fill_(~s["key_mask"][:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    safe = top.masked_fill(top == -math.inf, 0.0)
    p = score.sub_(safe).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2)) / total.masked_fill(total == 0, 1.0)
    lse = (safe + total.log()).view(B, H, L)
    out = out.view(B, G, H // G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H, D)
    return {"out": out.to(s["q"].dtype), "lse": lse}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, D = case["batch"], case["dim"]
    if case["op"] == "rotary":
        heads = case["q_heads"] + case["k_heads"]
        n = B * case["tokens"] * heads * D
        pos = (1 if case["shared"] else B) * case["tokens"] * _axes(case["grid"]) * 4
        return {"bytes": 2 * n * size + pos + case["rot"] // 2 * 4,
                "flops": (4 * n if case["norm"] else 0) + 3 * n * case["rot"] // D}
    L, S, H, G = case["q_tokens"], case["kv_tokens"], case["q_heads"], case["kv_heads"]
    if case["mask"] == "lens":
        read = sum(_lengths(case))
    elif case["mask"] == "pixels":
        kinds = {r: int(_valid_pixels(S, r).sum()) for r in set(_rects(case))}
        read = sum(kinds[r] for r in _rects(case))
    else:
        read = B * S
    mask = B * S if case["mask"] == "pixels" else 4 * B if case["mask"] == "lens" else 0
    return {"bytes": 2 * B * L * H * D * size + 4 * B * L * H + 2 * read * G * D * size + mask,
            "flops": 4 * read * L * H * D}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        rot, of = case["rot"], s["axis"]
        out = {}
        for n in ("q", "k"):
            if s[n] is None:
                continue
            x = s[n].double()
            if case["norm"]:
                x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt()
                x = x * s[n + "_weight"].double()
            # each pair as a complex number, turned by its angle
            lo = torch.arange(rot // 2, device=x.device)
            first, second = (2 * lo, 2 * lo + 1) if case["interleaved"] else (lo, lo + rot // 2)
            z = torch.complex(x[..., first], x[..., second])
            pos = torch.gather(s["positions"].double(), 2,
                               of.expand(*s["positions"].shape[:2], -1))
            z = z * torch.polar(torch.ones_like(pos), pos * s["freqs"].double())[:, :, None]
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[n] = y
        return out
    B, L, S = case["batch"], case["q_tokens"], case["kv_tokens"]
    H, G, D = case["q_heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(B, L, H, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, H, L), -math.inf, dtype=torch.float64, device=s["q"].device)
    for b in range(B):
        keep = torch.ones(S, dtype=torch.bool, device=s["q"].device)
        if s["kv_lens"] is not None:
            keep[int(s["kv_lens"][b]):] = False
        if s["key_mask"] is not None:
            keep &= s["key_mask"][b]
        if not bool(keep.any()):
            continue
        for h in range(H):
            k, v = (s[n][b, keep, h // (H // G)].double() for n in ("k", "v"))
            a = s["q"][b, :, h].double() @ k.T / math.sqrt(D)
            lse[b, h] = torch.logsumexp(a, -1)
            out[b, :, h] = torch.softmax(a, -1) @ v
    return {"out": out, "lse": lse}
