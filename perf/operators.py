"""The operators between a layer's QKV projection and its attention, and attention over a block-scaled cache:
what is timed, on which inputs, and what the answer is.

Three kinds of case, told apart by `kind`:

  rows    the queries' and keys' heads normed (RMS, 128 dims) and rotated to their positions
  append  the same on the way into a paged cache: keys rotated, then keys and values written into pages (fp16, E4M3
          with one scale per tensor, or E4M3 with one power-of-two scale per block of tokens and kv head)
  decode  one query token per sequence attending over a block-scaled E4M3 cache

A block is 16 tokens (8 where the page size is 8 modulo 16). Its K and V scales are bytes e that stand for 2^(e - 127),
the smallest in [2^-32, 2^8] with amax <= 448 scales; they only grow while a block fills.

Sequence lengths and places come from the case alone, values from the seed.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
D = 128           # head_dim
DEV = "cuda"
EPS = 1e-6
K_MIN, K_MAX = -32, 8   # exponents of block scales

own = False


def _pa():
    """This repository's package (imported only where `own` is true)."""
    if str(ROOT / "paged-attention_amd") not in sys.path:
        sys.path.insert(0, str(ROOT / "paged-attention_amd"))
    import pa_amd
    return pa_amd


def _rows(name, n, hq, hkv, rot=128, axes=1, interleaved=False, norm=True, fused=True, theta=500000.0):
    return {"name": name, "kind": "rows", "n": n, "hq": hq, "hkv": hkv, "rot": rot, "axes": axes,
            "interleaved": interleaved, "norm": norm, "fused": fused, "theta": theta, "far": 131072}


def _append(name, cache, batch, lo, hi, start, hq, hkv, page, rot=128, interleaved=False, norm=True, fused=True,
            theta=500000.0):
    return {"name": name, "kind": "append", "cache": cache, "batch": batch, "lo": lo, "hi": hi, "start": start,
            "hq": hq, "hkv": hkv, "page": page, "rot": rot, "axes": 1, "interleaved": interleaved, "norm": norm,
            "fused": fused, "theta": theta, "len_seed": 4}


def _decode(name, batch, lo, hi, hq, hkv, page):
    return {"name": name, "kind": "decode", "batch": batch, "lo": lo, "hi": hi, "hq": hq, "hkv": hkv, "page": page,
            "len_seed": 4}


def listed():
    return [
        # One new token of one sequence: launch latency only.
        _rows("rows 1 token", 1, 32, 8),
        # A long prompt's queries and keys, out of a fused projection.
        _rows("rows 8192 tokens", 8192, 32, 8),
        # Image and video tokens: time, height and width positions, interleaved pairs, an odd count, no head norm.
        _rows("rows 4999 tokens 3 axes", 4999, 16, 8, axes=3, interleaved=True, norm=False, fused=False, theta=10000.0),
        # A decode step of a busy server: one token of each of 64 sequences.
        _append("append step 64 fp16", "fp16", 64, 1, 1, 8192, 32, 8, 16),
        _append("append step 64 block", "block", 64, 1, 1, 8192, 32, 8, 16),
        # One long prompt into a quantized cache, with its queries.
        _append("append prompt 8192 fp8", "fp8", 1, 8192, 8192, 0, 32, 8, 16),
        # Ragged prompts that continue cached prefixes; half the dims rotated, a page size that is no power of two.
        _append("append 37 ragged block page 24", "block", 37, 1, 600, 900, 16, 4, 24, rot=64, theta=10000.0),
        # Several long prompts at once.
        _append("append 8x4096 block", "block", 8, 4096, 4096, 0, 32, 8, 16),
        # The smallest decode: one short chat turn.
        _decode("decode 1x200 block", 1, 200, 200, 32, 8, 16),
        # The headline batch at long context; the largest case.
        _decode("decode 64x8192 block", 64, 8192, 8192, 32, 8, 16),
        # Odd everything: lengths down to one token, 24-token pages, 8 query heads per kv head.
        _decode("decode 37 ragged block page 24", 37, 1, 3001, 64, 8, 24),
        # One long document: each sequence is cut over the whole chip.
        _decode("decode 1x131072 block", 1, 131072, 131072, 32, 8, 16),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rows", "append", "append", "decode"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 8), (8, 8), (4, 1), (8, 1), (16, 4), (6, 3)])
    theta = rng.choice([10000.0, 500000.0])
    rot, inter, norm, fused = rng.choice([128, 128, 64, 96, 32]), rng.random() < 0.4, rng.random() < 0.7, rng.random() < 0.6
    if kind == "rows":
        return {"kind": kind, "n": _log_int(rng, 1, 16384), "hq": hq, "hkv": hkv, "rot": rot,
                "axes": rng.choice([1, 1, 2, 3]), "interleaved": inter, "norm": norm, "fused": fused, "theta": theta,
                "far": _log_int(rng, 16, 1000000)}
    if kind == "append":
        cache = rng.choice(["fp16", "fp8", "block", "block"])
        page = rng.choice([8, 16, 16, 16, 24, 32, 64, 128] if cache == "block" else [1, 4, 16, 16, 24, 64, 100])
        batch = _log_int(rng, 1, 128)
        hi = 1 if rng.random() < 0.3 else _log_int(rng, 1, max(1, 20000 // batch))
        return {"kind": kind, "cache": cache, "batch": batch, "lo": hi if rng.random() < 0.4 else 1, "hi": hi,
                "start": rng.choice([0, _log_int(rng, 1, 20000)]), "hq": hq, "hkv": hkv, "page": page, "rot": rot,
                "axes": rng.choice([1, 1, 3]), "interleaved": inter, "norm": norm, "fused": fused, "theta": theta,
                "len_seed": rng.randrange(1000)}
    batch = _log_int(rng, 1, 128)
    hi = _log_int(rng, 16, min(131072, 262144 // batch))
    lo = hi if rng.random() < 0.4 else max(1, hi // rng.choice([2, 8, 1000]))
    return {"kind": kind, "batch": batch, "lo": lo, "hi": hi, "hq": hq if hq % 3 else 32, "hkv": hkv if hkv != 3 else 8,
            "page": rng.choice([8, 16, 16, 16, 24, 32, 64, 128]), "len_seed": rng.randrange(1000)}


def _lens(case: dict) -> list[int]:
    r = random.Random(case["len_seed"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _starts(case: dict) -> list[int]:
    r = random.Random(case["len_seed"] + 1)
    return [r.randint(case["start"] // 2, case["start"]) for _ in range(case["batch"])]


def _block(page: int) -> int:
    return 16 if page % 16 == 0 else 8


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(shape, g) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.float16, device=DEV).normal_(generator=g)


def _freqs(case: dict) -> list[float]:
    return [case["theta"] ** (-2.0 * i / case["rot"]) for i in range(case["rot"] // 2)]


def _axis_of(case: dict) -> list[int]:
    """Which of a token's positions turns pair i: runs of pairs, a quarter to time where there are three."""
    m, a = case["rot"] // 2, case["axes"]
    cut = [m] if a == 1 else [m // 2, m] if a == 2 else [m // 4, m // 4 + 3 * m // 8, m]
    return [next(j for j, c in enumerate(cut) if i < c) for i in range(m)]


def _heads(case: dict, n: int, g) -> dict:
    """A projection's output: q, k and v [n, heads, 128], views of one buffer where it is fused. Some channels of k
    are several times larger than the rest, as in trained models."""
    hq, hkv = case["hq"], case["hkv"]
    loud = torch.where(torch.arange(D, device=DEV) % 37 == 5, 6.0, 1.0).half()
    if case["fused"]:
        x = _normal((n, hq + 2 * hkv, D), g)
        x[:, hq:hq + hkv] *= loud
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    else:
        q, k, v = _normal((n, hq, D), g), _normal((n, hkv, D), g) * loud, _normal((n, hkv, D), g)
    w = [1.0 + 0.2 * torch.empty(D, device=DEV).normal_(generator=g) for _ in range(2)] if case["norm"] else [None, None]
    return {"q": q, "k": k, "v": v, "qw": w[0], "kw": w[1],
            "freqs": torch.tensor(_freqs(case), dtype=torch.float64, device=DEV),
            "axis_of": torch.tensor(_axis_of(case), device=DEV)}


def _rows_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    s = _heads(case, case["n"], g)
    s["pos"] = torch.randint(0, case["far"], (case["n"], case["axes"]), device=DEV, generator=g).to(torch.int32)
    return s


def _quantize_blocks(x: torch.Tensor):
    """x [..., tokens of a block, 128] as E4M3 codes and scale bytes: how a cache that was filled block by block lies."""
    _, e = torch.frexp(x.abs().amax(dim=(-1, -2)).float() / 448.0 * (1 - 2.0 ** -24))
    e = e.clamp(K_MIN, K_MAX)
    codes = torch.ldexp(x.float(), -e[..., None, None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _append_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    lens, starts, P, hkv = _lens(case), _starts(case), case["page"], case["hkv"]
    s = _heads(case, sum(lens), g)
    # Only the pages from the first new token's on are distinct: the call does not touch those before.
    first = [a // P for a in starts]
    last = [(a + n - 1) // P for a, n in zip(starts, lens)]
    count = torch.tensor([z - a + 1 for a, z in zip(first, last)])
    total = int(count.sum()) + 1
    perm = (torch.randperm(total - 1, device=DEV, generator=g) + 1).to(torch.int32)
    col = torch.arange(max(last) + 1, device=DEV)[None, :]
    fst, cnt = torch.tensor(first, device=DEV)[:, None], count.to(DEV)[:, None]
    at = (cnt.cumsum(0) - cnt + col - fst).clamp_(0, total - 2)
    # Image and video tokens have positions of their own; a text token's is its place in the cache.
    s["pos"] = None if case["axes"] == 1 else torch.randint(0, 4096, (sum(lens), case["axes"]), device=DEV,
                                                            generator=g).to(torch.int32)
    s["table"] = torch.where((col >= fst) & (col < fst + cnt), perm[at], 0).to(torch.int32).contiguous()
    s["tok_begin"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    s["starts"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
    shape = (total, hkv, P, D)
    s["scale"], s["scales"] = 1.0, None
    if case["cache"] == "fp16":
        s["kc"], s["vc"] = _normal(shape, g), _normal(shape, g)
    elif case["cache"] == "fp8":
        s["scale"] = 26.0 / 448.0
        s["kc"], s["vc"] = ((_normal(shape, g) * 40.0).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2))
    else:
        B = _block(P)
        pairs = [_quantize_blocks(_normal((total, hkv, P // B, B, D), g)) for _ in range(2)]
        s["kc"], s["vc"] = (c.view(shape) for c, _ in pairs)
        s["scales"] = torch.stack([e for _, e in pairs], dim=-1).contiguous()
    return s


def _decode_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    lens, P, hkv = _lens(case), case["page"], case["hkv"]
    B = _block(P)
    pages = [-(-n // P) for n in lens]
    total = sum(pages) + 3
    nbytes = total * hkv * P * D
    # One allocation, V a few KiB after the end of K: pools at the same offset modulo a large power of two would put
    # a page's K and V on the same memory banks.
    flat = torch.empty(2 * nbytes + 8192, dtype=torch.uint8, device=DEV)
    k, v = flat[:nbytes].view(total, hkv, P, D), flat[nbytes + 8192:].view(total, hkv, P, D)
    scales = torch.empty((total, hkv, P // B, 2), dtype=torch.uint8, device=DEV)
    chunk = max(1, (1 << 26) // (hkv * P * D))
    for i in range(0, total, chunk):
        for j, pool in enumerate((k, v)):
            n = min(chunk, total - i)
            loud = torch.exp2(torch.empty((n, hkv, P // B, 1, 1), device=DEV).uniform_(-2.0, 2.0, generator=g)).half()
            codes, e = _quantize_blocks(_normal((n, hkv, P // B, B, D), g) * loud)
            pool[i:i + n] = codes.view(n, hkv, P, D)
            scales[i:i + n, :, :, j] = e
    perm = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    first = torch.tensor([0] + pages[:-1]).cumsum(0).to(DEV)
    col = torch.arange(max(pages), device=DEV)
    at = (first[:, None] + col[None, :]).clamp_(max=total - 1)
    table = torch.where(col[None, :] < torch.tensor(pages, device=DEV)[:, None], perm[at], 0).to(torch.int32)
    return {"k": k, "v": v, "scales": scales, "table": table.contiguous(), "q": _normal((len(lens), case["hq"], D), g)}


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "rows":
        s = _rows_inputs(case, seed)
    elif case["kind"] == "append":
        s = _append_inputs(case, seed)
    else:
        s = _decode_inputs(case, seed)
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32)
        s["lens_dev"] = s["lens"].to(DEV)
    s["case"] = case
    if own:
        s["pa"] = _pa()
    if own and case["kind"] == "decode":   # a serving step plans once and runs every layer with that plan
        s["dec"] = s["pa"].Decoder(case["hq"], case["hkv"], D, case["page"], True, block_scales=True)
        s["dec"].plan(s["lens"])
    elif own:                              # a model's rotation, made once
        s["rope"] = s["pa"].Rope(_freqs(case), axes=_axis_of(case), interleaved=case["interleaved"])
    return s


def _norm_rotate(case: dict, x: torch.Tensor, w, pos: torch.Tensor, s: dict) -> torch.Tensor:
    """Heads x [n, h, 128] normed and rotated, in 32 bits (angles in 64): pos [n, axes]."""
    x, rot = x.float(), case["rot"]
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w
    angle = pos[:, s["axis_of"]].double() * s["freqs"]
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _need(amax: torch.Tensor) -> torch.Tensor:
    """The smallest k in range with amax <= 448 * 2^k."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875), K_MIN).clamp(K_MIN, K_MAX)


def _encode(x: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """E4M3 of x / 2^k, saturated at 448 (240 where k is the largest: no fp16 lies above 61440 with four bits)."""
    top = torch.where(k == K_MAX, 240.0, 448.0)
    return torch.maximum(torch.minimum(torch.ldexp(x, -k), top), -top).to(torch.float8_e4m3fn).view(torch.uint8)


def _append_blocks(pool: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, page, slot, s: dict, B: int) -> None:
    """Rows x [n, hkv, 128] at (page, slot) of a block-scaled pool; scales [pages, hkv, blocks of a page]."""
    total, hkv, P, _ = pool.shape
    nb, blk, t0 = P // B, slot // B, s["starts"].long()
    # What each block has to hold of this call, and whether it begins with it.
    flat = (page * nb + blk)[:, None].expand(-1, hkv)
    amax = torch.zeros((total * nb, hkv), device=DEV).scatter_reduce(0, flat, x.abs().amax(dim=-1), "amax")
    fresh = torch.zeros(total * nb, dtype=torch.int32, device=DEV)
    fresh = fresh.scatter_reduce(0, page * nb + blk, (slot % B == 0).int(), "amax").bool()
    touched = torch.zeros(total * nb, dtype=torch.bool, device=DEV).index_fill(0, page * nb + blk, True)
    old = scales.permute(0, 2, 1).reshape(total * nb, hkv).int() - 127
    need = _need(amax)
    new = torch.where(fresh[:, None], need, torch.maximum(old, need))
    new = torch.where(touched[:, None], new, old)
    scales.copy_((new + 127).to(torch.uint8).view(total, nb, hkv).permute(0, 2, 1))
    # The first block of each sequence may hold earlier rows: to their block's new scale.
    p0 = s["table"].gather(1, (t0 // P)[:, None])[:, 0].long()
    b0 = t0 % P // B
    view = pool.view(total, hkv, nb, B, D)
    held = view[p0, :, b0]
    at = p0 * nb + b0
    moved = _encode(torch.ldexp(held.view(torch.float8_e4m3fn).float(), old[at][..., None, None]), new[at][..., None, None])
    earlier = torch.arange(B, device=DEV)[None, :] < (t0 % B)[:, None]
    grown = (new[at] > old[at])[..., None, None]
    view[p0, :, b0] = torch.where(earlier[:, None, :, None] & grown, moved, held)
    pool[page, :, slot] = _encode(x, new[page * nb + blk][..., None])


def _append_plain(case: dict, s: dict):
    P, n = case["page"], s["k"].shape[0]
    t = torch.arange(n, device=DEV, dtype=torch.int32)
    e = torch.searchsorted(s["tok_begin"], t, right=True) - 1
    pos = (s["starts"][e] + t - s["tok_begin"][e]).long()
    page, slot = s["table"][e, pos // P].long(), pos % P
    turn = pos[:, None] if s["pos"] is None else s["pos"]
    q = _norm_rotate(case, s["q"], s["qw"], turn, s).half()
    k, v = _norm_rotate(case, s["k"], s["kw"], turn, s), s["v"].float()
    if case["cache"] == "block":
        B = _block(P)
        _append_blocks(s["kc"], s["scales"][..., 0], k, page, slot, s, B)
        _append_blocks(s["vc"], s["scales"][..., 1], v, page, slot, s, B)
    elif case["cache"] == "fp8":
        inv = torch.tensor(1.0, device=DEV) / s["scale"]
        s["kc"][page, :, slot] = (k * inv).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        s["vc"][page, :, slot] = (v * inv).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["kc"][page, :, slot] = k.half()
        s["vc"][page, :, slot] = s["v"]
    return q


def _decode_plain(s: dict, case: dict):
    """Every row padded to the longest: scores of the pages' tokens, masked behind each row's length."""
    P, hkv, hq = case["page"], case["hkv"], case["hq"]
    rows, cols = s["table"].shape
    index = s["table"].long().view(-1)
    factor = torch.exp2(s["scales"].float() - 127.0).repeat_interleave(_block(P), dim=2)[index]

    def kept(pool, j):
        x = pool[index].view(torch.float8_e4m3fn).float() * factor[..., j, None]
        return x.view(rows, cols, hkv, P, D).transpose(1, 2).reshape(rows, hkv, cols * P, D)
    qt = s["q"].float().view(rows, hkv, hq // hkv, D).transpose(2, 3).contiguous()
    w = torch.matmul(kept(s["k"], 0), qt) / math.sqrt(D)
    behind = torch.arange(cols * P, device=DEV)[None, :] >= s["lens_dev"][:, None]
    w = w.masked_fill_(behind[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(dim=2, keepdim=True))
    w = (w / w.sum(dim=2, keepdim=True)).transpose(2, 3).contiguous()
    return torch.matmul(w, kept(s["v"], 1)).half().view(rows, hq, D)


def run(s: dict):
    case = s["case"]
    if case["kind"] == "rows":
        if own:
            return s["pa"].norm_rope(s["q"], s["k"], s["pos"], s["rope"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
        return tuple(_norm_rotate(case, x, w, s["pos"], s).half() for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
    if case["kind"] == "append":
        if own:
            q = s["pa"].append_rope(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["tok_begin"], s["starts"],
                                    s["rope"], positions=s["pos"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                    k_scale=s["scale"], v_scale=s["scale"], kv_scales=s["scales"])
        else:
            q = _append_plain(case, s)
        if case["cache"] == "fp16":
            return q, s["kc"], s["vc"]
        out = q, s["kc"].view(torch.float8_e4m3fn), s["vc"].view(torch.float8_e4m3fn)
        return out if s["scales"] is None else out + (s["scales"].view(torch.float8_e8m0fnu),)
    if own:
        return s["dec"].run(s["q"], s["k"], s["v"], s["table"], s["lens_dev"], 1.0, 1.0, kv_scales=s["scales"])
    return _decode_plain(s, case)


def work(case: dict) -> dict:
    hq, hkv = case["hq"], case["hkv"]
    if case["kind"] == "decode":
        n = sum(_lens(case))
        blocks = sum(-(-x // _block(case["page"])) for x in _lens(case))
        kv = 2 * n * hkv * D + 2 * blocks * hkv + 4 * sum(-(-x // case["page"]) for x in _lens(case))
        return {"bytes": kv + 4 * case["batch"] * hq * D, "flops": 4 * n * hq * D}
    n = case["n"] if case["kind"] == "rows" else sum(_lens(case))
    turned = n * (hq + hkv)
    if case["kind"] == "rows":
        return {"bytes": 4 * turned * D + 4 * n * case["axes"], "flops": 7 * turned * D}
    out = 2 if case["cache"] == "fp16" else 1
    scales = 2 * hkv * (n // 16 + case["batch"]) if case["cache"] == "block" else 0
    return {"bytes": 4 * n * hq * D + 2 * n * hkv * D * (2 + out) + scales + 12 * case["batch"] + 4 * (n // case["page"])
            + (4 * n * case["axes"] if case["axes"] > 1 else 0), "flops": 7 * turned * D}


def _turn64(case: dict, x: torch.Tensor, w, pos: torch.Tensor) -> torch.Tensor:
    """The definition in 64 bits, as a product of complex numbers: x [n, h, 128], pos [n, axes]."""
    x, m = x.double(), case["rot"] // 2
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    f = torch.tensor(_freqs(case), dtype=torch.float64, device=DEV)
    axis = torch.tensor(_axis_of(case), device=DEV)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[:, axis] * f)[:, None]
    out = x.clone()
    if case["interleaved"]:
        z = torch.complex(x[..., :2 * m].unflatten(-1, (m, 2))[..., 0], x[..., :2 * m].unflatten(-1, (m, 2))[..., 1]) * turn
        out[..., :2 * m] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :m], x[..., m:2 * m]) * turn
        out[..., :m], out[..., m:2 * m] = z.real, z.imag
    return out


def _exact_append(case: dict, seed: int):
    s = _append_inputs(case, seed)
    lens, starts, P, hkv = _lens(case), _starts(case), case["page"], case["hkv"]
    pos = torch.cat([torch.arange(a, a + n, device=DEV) for a, n in zip(starts, lens)])
    turn = pos[:, None] if s["pos"] is None else s["pos"]
    q, k = (_turn64(case, x, w, turn) for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
    pools, scales = [], []
    for j, (pool, x) in enumerate(((s["kc"], k), (s["vc"], s["v"].double()))):
        held = pool.double() if case["cache"] == "fp16" else pool.view(torch.float8_e4m3fn).double()
        exps = None if s["scales"] is None else s["scales"][..., j].double() - 127.0
        at = 0
        for b, (a, n) in enumerate(zip(starts, lens)):
            p = torch.arange(a, a + n, device=DEV)
            page, slot, part = s["table"][b, p // P].long(), p % P, x[at:at + n]
            at += n
            if case["cache"] == "block":
                B = _block(P)
                # Per block of this sequence: the largest value, by runs of tokens that lie in it.
                order, run_of, _ = torch.unique_consecutive(p // B, return_inverse=True, return_counts=True)
                big = torch.zeros((len(order), hkv), dtype=torch.float64, device=DEV)
                big = big.scatter_reduce(0, run_of[:, None].expand(-1, hkv), part.abs().amax(-1), "amax")
                need = torch.ceil(torch.log2(big / 448.0)).clamp(K_MIN, K_MAX)
                first = order * B
                pg, bk = s["table"][b, first // P].long(), first % P // B
                old = exps[pg, :, bk]
                if a % B:
                    need[0] = torch.maximum(need[0], old[0])
                    rows = held[pg[0], :, int(first[0]) % P:int(first[0]) % P + a % B]
                    rows *= torch.exp2(old[0] - need[0])[:, None, None]
                exps[pg, :, bk] = need
                held[page, :, slot] = part * torch.exp2(-need[run_of])[..., None]
            else:
                held[page, :, slot] = part / s["scale"]
        pools.append(held)
        scales.append(exps)
    out = (q, pools[0], pools[1])
    return out if s["scales"] is None else out + (torch.exp2(torch.stack(scales, dim=-1)),)


def _exact_decode(case: dict, seed: int):
    s = _decode_inputs(case, seed)
    P, hkv, B, out = case["page"], case["hkv"], _block(case["page"]), []
    for b, n in enumerate(_lens(case)):
        pages = s["table"][b, :-(-n // P)].long()
        kv = []
        for j, pool in enumerate((s["k"], s["v"])):
            x = pool[pages].view(torch.float8_e4m3fn).double().view(-1, hkv, P // B, B, D)
            x = x * torch.exp2(s["scales"][pages][..., j].double() - 127.0)[..., None, None]
            kv.append(x.view(-1, hkv, P, D).transpose(0, 1).reshape(hkv, -1, D)[:, :n].contiguous())
        score = torch.matmul(s["q"][b].double().view(hkv, -1, D), kv[0].transpose(1, 2).contiguous()) / math.sqrt(D)
        out.append(torch.matmul(torch.softmax(score, dim=-1), kv[1]).reshape(-1, D))
    return torch.stack(out)


def exact(case: dict, seed: int):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "decode":
        return _exact_decode(case, seed)
    s = _rows_inputs(case, seed)
    return tuple(_turn64(case, x, w, s["pos"]) for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
