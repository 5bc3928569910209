"""Drafted tokens over a paged cache: what is timed, on which inputs, and what the answer is.

Three kinds of case, told apart by `kind`:

  attend  several new tokens per sequence, stored in the cache behind it, attend over it: every token sees its
          sequence's earlier places and, of the new ones, those that its row of a tree names (`tree`), or itself
          and those before it (a chain: a prompt's piece, or a draft without branches)
  keep    of a sequence's drafted tokens those that were accepted move up in the cache, in place
  read    places of several sequences read back from the pages, side by side, in a type to compute with

Caches hold fp16, E4M3 with one scale per tensor (fp8), or E4M3 with a power-of-two scale per block of tokens and kv
head (block): 16 tokens (8 where the page size is 8 modulo 16), bytes e for 2^(e - 127), K's and V's side by side,
the smallest in [2^-32, 2^8] with amax <= 448 scales.

Lengths, places and types come from the case alone, values, trees and accepted tokens from the seed.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
D = 128                 # head_dim
DEV = "cuda"
K_MIN, K_MAX = -32, 8   # exponents of block scales
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

own = False


def _pa():
    """This repository's package (imported only where `own` is true)."""
    if str(ROOT / "paged-attention_amd") not in sys.path:
        sys.path.insert(0, str(ROOT / "paged-attention_amd"))
    import pa_amd
    return pa_amd


def _attend(name, cache, batch, lo, hi, drafts, hq, hkv, page, tree=True, ragged=False):
    """batch sequences of lo .. hi earlier places, each with `drafts` new tokens (1 .. drafts if ragged)."""
    return {"name": name, "kind": "attend", "cache": cache, "batch": batch, "lo": lo, "hi": hi, "drafts": drafts,
            "ragged": ragged, "hq": hq, "hkv": hkv, "page": page, "tree": tree, "len_seed": 4}


def _keep(name, cache, batch, start, drafts, most, hkv, page):
    return {"name": name, "kind": "keep", "cache": cache, "batch": batch, "start": start, "drafts": drafts,
            "most": most, "hkv": hkv, "page": page, "len_seed": 4}


def _read(name, cache, batch, lo, hi, start, hkv, page, out="fp16"):
    return {"name": name, "kind": "read", "cache": cache, "batch": batch, "lo": lo, "hi": hi, "start": start,
            "hkv": hkv, "page": page, "out": out, "len_seed": 4}


def listed():
    return [
        # One short chat turn with a small tree: launch latency.
        _attend("tree 8 over 1x200 fp16", "fp16", 1, 200, 200, 8, 32, 8, 16),
        # The headline batch verifying a tree at each sequence.
        _attend("tree 16 over 32x8192 fp16", "fp16", 32, 8192, 8192, 16, 32, 8, 16),
        # The block-scaled batch with wide trees: as much arithmetic as memory traffic.
        _attend("tree 32 over 64x8192 block", "block", 64, 8192, 8192, 32, 32, 8, 16),
        # One long document, one scale per tensor: a sequence is cut over the whole chip.
        _attend("tree 64 over 1x131072 fp8", "fp8", 1, 131072, 131072, 64, 32, 8, 16),
        # Odd everything: lengths down to one token, 24-token pages, 8 query heads per kv head, ragged drafts.
        _attend("tree 1-60 over 37 ragged block page 24", "block", 37, 1, 3001, 60, 64, 8, 24, ragged=True),
        # A long prompt's second piece over its first: arithmetic only.
        _attend("chain 4096 over 4096 fp16", "fp16", 1, 4096, 4096, 4096, 32, 8, 16, tree=False),
        # What of a busy server's drafts was accepted.
        _keep("keep 64 of 32 fp16", "fp16", 64, 8192, 32, 6, 8, 16),
        _keep("keep 64 of 32 block", "block", 64, 8192, 32, 6, 8, 16),
        # A large batch's, wide trees with long paths.
        _keep("keep 512 of 64 fp8", "fp8", 512, 2000, 64, 16, 8, 16),
        # A short prefix back from the cache: latency.
        _read("read 1x100 block", "block", 1, 100, 100, 0, 8, 16),
        # Ragged prefixes from odd places and pages.
        _read("read 37 ragged fp8 page 24", "fp8", 37, 1, 3001, 900, 8, 24, "bf16"),
        # Long prefixes of several sequences.
        _read("read 8x8192 block", "block", 8, 8192, 8192, 0, 8, 16),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "keep", "read"])
    cache = rng.choice(["fp16", "fp8", "block"])
    page = rng.choice([8, 16, 16, 16, 24, 32, 64, 128] if cache == "block" else [1, 4, 16, 16, 24, 64, 100])
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 8), (8, 8), (4, 1), (8, 1), (16, 4), (6, 3), (9, 3)])
    seed = rng.randrange(1000)
    if kind == "attend":
        tree = rng.random() < 0.65
        batch = _log_int(rng, 1, 128)
        drafts = _log_int(rng, 1, 100) if tree else _log_int(rng, 1, max(1, min(4096, 131072 // hq) // batch))
        # No more cached bytes than the headline batch, no more products than the largest listed case.
        most = min(131072, 262144 // batch, max(16, (1 << 29) // (batch * drafts * hq)))
        hi = _log_int(rng, 16, most)
        lo = hi if rng.random() < 0.4 else max(1, hi // rng.choice([2, 8, 1000]))
        if rng.random() < 0.1:
            lo = hi = 0
        return {"kind": kind, "cache": cache, "batch": batch, "lo": lo, "hi": hi, "drafts": drafts,
                "ragged": rng.random() < 0.5, "hq": hq, "hkv": hkv, "page": page, "tree": tree, "len_seed": seed}
    batch = _log_int(rng, 1, 512)
    if kind == "keep":
        drafts = _log_int(rng, 1, 100)
        return {"kind": kind, "cache": cache, "batch": batch, "start": rng.choice([0, _log_int(rng, 1, 20000)]),
                "drafts": drafts, "most": rng.randint(1, drafts), "hkv": hkv, "page": page, "len_seed": seed}
    hi = _log_int(rng, 1, max(1, 65536 // batch))
    return {"kind": kind, "cache": cache, "batch": batch, "lo": hi if rng.random() < 0.4 else 1, "hi": hi,
            "start": rng.choice([0, _log_int(rng, 1, 5000)]), "hkv": hkv, "page": page,
            "out": rng.choice(["fp16", "fp16", "bf16", "fp32"]), "len_seed": seed}


def _between(case: dict, lo: int, hi: int, salt: int = 0) -> list[int]:
    r = random.Random(case["len_seed"] + salt)
    return [r.randint(lo, hi) for _ in range(case["batch"])]


def _drafts(case: dict) -> list[int]:
    return _between(case, 1 if case["ragged"] else case["drafts"], case["drafts"], 1)


def _counts(case: dict) -> list[int]:
    return _between(case, 1, case["most"], 2)


def _starts(case: dict) -> list[int]:
    """First place that is new (attend, keep) or read."""
    if case["kind"] == "attend":
        return _between(case, case["lo"], case["hi"])
    return _between(case, case["start"] // 2, case["start"], 1)


def _ends(case: dict) -> list[int]:
    new = (_drafts(case) if case["kind"] == "attend" else [case["drafts"]] * case["batch"] if case["kind"] == "keep"
           else _between(case, case["lo"], case["hi"]))
    return [a + n for a, n in zip(_starts(case), new)]


def _block(page: int) -> int:
    return 16 if page % 16 == 0 else 8


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32).to(DEV)


def _quantize_blocks(x: torch.Tensor):
    """x [..., tokens of a block, 128] as E4M3 codes and scale bytes: how a cache that was filled block by block lies."""
    _, e = torch.frexp(x.abs().amax(dim=(-1, -2)).float() / 448.0 * (1 - 2.0 ** -24))
    e = e.clamp(K_MIN, K_MAX)
    codes = torch.ldexp(x.float(), -e[..., None, None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _inputs(case: dict, seed: int) -> dict:
    """Caches, tables and places. Pages before the first that the call touches are not made (`keep`, `read`)."""
    g = _gen(seed)
    P, hkv, cache = case["page"], case["hkv"], case["cache"]
    starts, ends = _starts(case), _ends(case)
    first = [0] * len(starts) if case["kind"] == "attend" else [a // P for a in starts]
    last = [(z - 1) // P for z in ends]
    count = torch.tensor([z - a + 1 for a, z in zip(first, last)])
    total = int(count.sum()) + 3
    perm = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    col = torch.arange(max(last) + 1, device=DEV)[None, :]
    fst, cnt = torch.tensor(first, device=DEV)[:, None], count.to(DEV)[:, None]
    at = (cnt.cumsum(0) - cnt + col - fst).clamp_(0, total - 1)
    s = {"table": torch.where((col >= fst) & (col < fst + cnt), perm[at], 0).to(torch.int32).contiguous(),
         "starts": _ints(starts), "scales": None, "kscale": 1.0, "vscale": 1.0}
    elem = 2 if cache == "fp16" else 1
    nbytes = total * hkv * P * D * elem
    # One allocation, V a few KiB after the end of K: pools at the same offset modulo a large power of two would put
    # a page's K and V on the same memory banks.
    flat = torch.empty(2 * nbytes + 8192, dtype=torch.uint8, device=DEV)
    shape = (total, hkv, P, D)
    pools = [flat[o:o + nbytes].view(torch.float16 if elem == 2 else torch.uint8).view(shape) for o in (0, nbytes + 8192)]
    if cache == "block":
        s["scales"] = torch.empty((total, hkv, P // _block(P), 2), dtype=torch.uint8, device=DEV)
    if cache == "fp8":
        s["kscale"], s["vscale"] = 5.0 / 448.0, 6.0 / 448.0
    B, chunk = _block(P), max(1, (1 << 26) // (hkv * P * D))
    for i in range(0, total, chunk):
        n = min(chunk, total - i)
        for j, pool in enumerate(pools):
            if cache == "fp16":
                pool[i:i + n].normal_(generator=g)
            elif cache == "fp8":
                x = torch.empty((n, hkv, P, D), dtype=torch.float16, device=DEV).normal_(generator=g)
                pool[i:i + n] = (x.float() / s["vscale" if j else "kscale"]).clamp_(-448.0, 448.0).to(
                    torch.float8_e4m3fn).view(torch.uint8)
            else:
                loud = torch.exp2(torch.empty((n, hkv, P // B, 1, 1), device=DEV).uniform_(-2.0, 2.0, generator=g))
                x = torch.empty((n, hkv, P // B, B, D), dtype=torch.float16, device=DEV).normal_(generator=g)
                codes, e = _quantize_blocks(x * loud.half())
                pool[i:i + n] = codes.view(n, hkv, P, D)
                s["scales"][i:i + n, :, :, j] = e
    s["kc"], s["vc"] = pools
    if case["kind"] == "attend":
        new = _drafts(case)
        s["tok_begin"] = _ints([0] + new).cumsum(0).to(torch.int32)
        s["q"] = torch.empty((sum(new), case["hq"], D), dtype=torch.float16, device=DEV).normal_(generator=g).mul_(2.0)
        s["tree"] = _trees(case, seed) if case["tree"] else None
    elif case["kind"] == "keep":
        s["kept"], s["counts"] = _ints(_paths(case, seed)), _ints(_counts(case))
    else:
        s["tok_begin"] = _ints([0] + [z - a for a, z in zip(starts, ends)]).cumsum(0).to(torch.int32)
        s["n"] = sum(ends) - sum(starts)
    return s


def _rows_of_trees(case: dict, seed: int) -> list[list[int]]:
    """For each sequence its drafted tokens' rows: the token itself, what it continues, and so on up to token 0, which
    continues the sequence; whole numbers whose bit j is token j."""
    r = random.Random(seed)
    out = []
    for n in _drafts(case):
        rows: list[int] = []
        for i in range(n):
            rows.append((1 << i) | (rows[r.randrange(max(0, i - 12), i)] if i else 0))
        out.append(rows)
    return out


def _trees(case: dict, seed: int) -> torch.Tensor:
    words = -(-case["drafts"] // 64)
    flat = [(row >> (64 * w)) & (2 ** 64 - 1) for rows in _rows_of_trees(case, seed) for row in rows for w in range(words)]
    return torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in flat], dtype=torch.int64).view(-1, words).to(DEV)


def _paths(case: dict, seed: int) -> list[list[int]]:
    """Per sequence the accepted tokens, rising, padded to the longest path; token 0 continues the sequence."""
    r = random.Random(seed)
    return [sorted([0] + r.sample(range(1, case["drafts"]), n - 1)) + [0] * (case["most"] - n) for n in _counts(case)]


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["pa"] = _pa()
    return s


def _values(case: dict, s: dict, pool: torch.Tensor, j: int, page: torch.Tensor, slot: torch.Tensor) -> torch.Tensor:
    """Rows [..., hkv, 128] of a pool (j: 0 keys, 1 values) at page and slot, as the numbers that they stand for."""
    x = pool[page, :, slot]
    if case["cache"] == "fp16":
        return x.float()
    x = x.view(torch.float8_e4m3fn).float()
    if case["cache"] == "fp8":
        return x * s["vscale" if j else "kscale"]
    return x * torch.exp2(s["scales"][..., j][page, :, slot // _block(case["page"])].float() - 127.0)[..., None]


def _attend_plain(case: dict, s: dict) -> torch.Tensor:
    """Every sequence padded to the longest, in tokens and places: scores, masked, their softmax, the values' sum."""
    P, hq, hkv, batch = case["page"], case["hq"], case["hkv"], case["batch"]
    n, tb, start = s["q"].shape[0], s["tok_begin"].long(), s["starts"].long()
    new = tb[1:] - tb[:-1]
    T, places = case["drafts"], s["table"].shape[1] * P
    at = torch.arange(places, device=DEV)
    page = s["table"].long()[:, at // P]
    kv = [_values(case, s, pool, j, page, (at % P).expand(batch, -1)).transpose(1, 2).contiguous()
          for j, pool in enumerate((s["kc"], s["vc"]))]
    tok = torch.arange(T, device=DEV)
    t = (tb[:-1, None] + tok).clamp_(max=n - 1)                                       # [batch, T]
    rel = at[None, :] - start[:, None]                                                # [batch, places]
    if s["tree"] is None:
        seen = rel[:, None, :] <= tok[None, :, None]
    else:
        word = s["tree"][t]                                                           # [batch, T, words]
        bit = rel.clamp(0, 64 * word.shape[2] - 1)
        pick = torch.gather(word, 2, (bit // 64)[:, None, :].expand(-1, T, -1))
        seen = (rel[:, None, :] < 0) | ((pick >> (bit % 64)[:, None, :]) & 1).bool()
    seen = seen & (rel < new[:, None])[:, None, :]
    q = s["q"][t].float().view(batch, T, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, D)
    w = torch.matmul(q, kv[0].transpose(2, 3).contiguous()) / math.sqrt(D)            # [batch, hkv, T * group, places]
    w = w.view(batch, hkv, T, -1, places).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = w.amax(dim=-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    w = w.div_(w.sum(dim=-1, keepdim=True).clamp_min_(1e-30)).view(batch, hkv, -1, places)
    out = torch.matmul(w, kv[1]).half().view(batch, hkv, T, -1, D).permute(0, 2, 1, 3, 4).reshape(batch, T, hq, D)
    e = torch.searchsorted(tb[1:].contiguous(), torch.arange(n, device=DEV), right=True)
    return out[e, torch.arange(n, device=DEV) - tb[e]]


def _need(amax: torch.Tensor) -> torch.Tensor:
    """The smallest k in range with amax <= 448 * 2^k."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875), K_MIN).clamp(K_MIN, K_MAX)


def _encode(x: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """E4M3 of x / 2^k, saturated at 448 (240 where k is the largest: no fp16 lies above 61440 with four bits)."""
    top = torch.where(k == K_MAX, 240.0, 448.0)
    return torch.maximum(torch.minimum(torch.ldexp(x, -k), top), -top).to(torch.float8_e4m3fn).view(torch.uint8)


def _keep_plain(case: dict, s: dict) -> None:
    P, hkv, most = case["page"], case["hkv"], s["kept"].shape[1]
    start = s["starts"].long()
    # Past an entry's count its first token again, which stays where it is or goes where it went.
    j = torch.arange(most, device=DEV)[None, :].expand(case["batch"], -1)
    live = j < s["counts"][:, None]
    j = torch.where(live, j, 0)
    src = start[:, None] + torch.gather(s["kept"].long(), 1, j)
    dst = start[:, None] + j
    table = s["table"].long()
    ps, pd = torch.gather(table, 1, src // P).view(-1), torch.gather(table, 1, dst // P).view(-1)
    ss, sd = (src % P).view(-1), (dst % P).view(-1)
    if case["cache"] != "block":
        for pool in (s["kc"], s["vc"]):
            pool[pd, :, sd] = pool[ps, :, ss]
        return
    B = _block(P)
    total, nb = s["kc"].shape[0], P // B
    home = pd * nb + sd // B                                                    # the block that a row comes to
    moved = torch.zeros(total * nb, dtype=torch.int32, device=DEV).scatter_reduce(0, home, (src != dst).view(-1).int(),
                                                                                  "amax").bool()
    fresh = torch.zeros(total * nb, dtype=torch.int32, device=DEV).scatter_reduce(
        0, home, (dst // B * B >= start[:, None]).view(-1).int(), "amax").bool()
    p0, b0 = torch.gather(table, 1, (start // P)[:, None])[:, 0], start % P // B
    at = p0 * nb + b0                                                           # the block that may hold earlier rows
    for i, pool in enumerate((s["kc"], s["vc"])):
        x = _values(case, s, pool, i, ps, ss)                                   # [rows, hkv, 128]
        amax = torch.zeros((total * nb, hkv), device=DEV).scatter_reduce(
            0, home[:, None].expand(-1, hkv), x.abs().amax(dim=-1), "amax")
        scales = s["scales"][..., i]
        old = scales.permute(0, 2, 1).reshape(total * nb, hkv).int() - 127
        now = torch.where(fresh[:, None], _need(amax), torch.maximum(old, _need(amax)))
        now = torch.where(moved[:, None], now, old)
        scales.copy_((now + 127).to(torch.uint8).view(total, nb, hkv).permute(0, 2, 1))
        view = pool.view(total, hkv, nb, B, D)
        held = view[p0, :, b0]
        to = _encode(torch.ldexp(held.view(torch.float8_e4m3fn).float(), old[at][..., None, None]), now[at][..., None, None])
        earlier = torch.arange(B, device=DEV)[None, :] < (start % B)[:, None]
        view[p0, :, b0] = torch.where(earlier[:, None, :, None] & (now[at] > old[at])[..., None, None], to, held)
        codes = _encode(x, now[home][..., None])
        pool[pd, :, sd] = torch.where(moved[home][:, None, None], codes, pool[pd, :, sd])


def _read_plain(case: dict, s: dict):
    t, tb = torch.arange(s["n"], device=DEV), s["tok_begin"].long()
    e = torch.searchsorted(tb, t, right=True) - 1
    pos = s["starts"].long()[e] + t - tb[e]
    page, slot = s["table"].long()[e, pos // case["page"]], pos % case["page"]
    return tuple(_values(case, s, pool, j, page, slot).to(TYPES[case["out"]]) for j, pool in enumerate((s["kc"], s["vc"])))


def _caches(case: dict, s: dict):
    if case["cache"] == "fp16":
        return s["kc"], s["vc"]
    out = s["kc"].view(torch.float8_e4m3fn), s["vc"].view(torch.float8_e4m3fn)
    return out if s["scales"] is None else out + (s["scales"].view(torch.float8_e8m0fnu),)


def run(s: dict):
    case = s["case"]
    if case["kind"] == "attend":
        if own:
            return s["pa"].tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["tok_begin"], s["starts"], s["tree"],
                                          k_scale=s["kscale"], v_scale=s["vscale"], kv_scales=s["scales"])
        return _attend_plain(case, s)
    if case["kind"] == "keep":
        if own:
            s["pa"].keep_rows(s["kc"], s["vc"], s["table"], s["kept"], s["counts"], s["starts"], kv_scales=s["scales"])
        else:
            _keep_plain(case, s)
        return _caches(case, s)
    if own:
        return s["pa"].read_cache(s["kc"], s["vc"], s["table"], s["tok_begin"], s["starts"], s["n"],
                                  dtype=TYPES[case["out"]], k_scale=s["kscale"], v_scale=s["vscale"],
                                  kv_scales=s["scales"])
    return _read_plain(case, s)


def work(case: dict) -> dict:
    hkv, P = case["hkv"], case["page"]
    row = 2 * hkv * D * (2 if case["cache"] == "fp16" else 1)   # a place's keys and values
    starts, ends = _starts(case), _ends(case)
    tables = sum(4 * (z // P - a // P + 1) for a, z in zip(starts, ends))
    if case["kind"] == "attend":
        new, hq = _drafts(case), case["hq"]
        scales = sum(2 * hkv * -(-z // _block(P)) for z in ends) if case["cache"] == "block" else 0
        # A chain's token sees half of the new ones; a tree's is taken to see them all (its products are masked).
        pairs = sum(n * a + (n * n if case["tree"] else n * (n + 1) // 2) for n, a in zip(new, starts))
        return {"bytes": row * sum(ends) + scales + sum(4 * -(-z // P) for z in ends) + 4 * sum(new) * hq * D
                + (8 * sum(new) * -(-case["drafts"] // 64) if case["tree"] else 0), "flops": 4 * pairs * hq * D}
    if case["kind"] == "keep":
        # What moves: a path's first token is in its place, hardly any later one is.
        n = sum(_counts(case)) - case["batch"]
        scales = 4 * hkv * 2 * case["batch"] if case["cache"] == "block" else 0
        return {"bytes": 2 * row * n + scales + 4 * n + 16 * case["batch"], "flops": 0}
    n = sum(ends) - sum(starts)
    scales = 2 * hkv * (n // _block(P) + case["batch"]) if case["cache"] == "block" else 0
    return {"bytes": n * (row + 2 * hkv * D * (4 if case["out"] == "fp32" else 2)) + scales + tables
            + 12 * case["batch"], "flops": n * 2 * hkv * D}


def _exact_kv(case: dict, s: dict, b: int, lo: int, hi: int):
    """Keys and values of places lo .. hi - 1 of sequence b in 64 bits, [hkv, places, 128] each."""
    P, hkv = case["page"], case["hkv"]
    pages = s["table"][b, lo // P:(hi - 1) // P + 1].long()
    out = []
    for j, pool in enumerate((s["kc"], s["vc"])):
        x = pool[pages]
        if case["cache"] == "fp16":
            x = x.double()
        elif case["cache"] == "fp8":
            x = x.view(torch.float8_e4m3fn).double() * s["vscale" if j else "kscale"]
        else:
            e = s["scales"][pages][..., j].double() - 127.0
            x = (x.view(torch.float8_e4m3fn).double().view(-1, hkv, P // _block(P), _block(P) * D)
                 * torch.exp2(e)[..., None]).view(-1, hkv, P, D)
        out.append(x.transpose(0, 1).reshape(hkv, -1, D)[:, lo % P:lo % P + hi - lo].contiguous())
    return out


def _exact_attend(case: dict, seed: int):
    s = _inputs(case, seed)
    hkv, group, out, at = case["hkv"], case["hq"] // case["hkv"], [], 0
    rows = _rows_of_trees(case, seed) if case["tree"] else None
    for b, (a, n) in enumerate(zip(_starts(case), _drafts(case))):
        k, v = _exact_kv(case, s, b, 0, a + n)
        if rows is None:
            seen = torch.ones((n, n), dtype=torch.bool, device=DEV).tril()
        else:
            seen = torch.tensor([[(row >> j) & 1 for j in range(n)] for row in rows[b]], dtype=torch.bool).to(DEV)
        hide = torch.cat([torch.zeros((n, a), dtype=torch.bool, device=DEV), ~seen], dim=1)
        q = s["q"][at:at + n].double().view(n, hkv, group, D)
        at += n
        o = torch.empty((n, hkv, group, D), dtype=torch.float64, device=DEV)
        for h in range(hkv):
            for g in range(group):
                x = torch.matmul(q[:, h, g].contiguous(), k[h].t().contiguous()) / math.sqrt(D)
                o[:, h, g] = torch.matmul(torch.softmax(x.masked_fill_(hide, -math.inf), dim=-1), v[h])
        out.append(o.view(n, -1, D))
    return torch.cat(out)


def _exact_keep(case: dict, seed: int):
    s = _inputs(case, seed)
    P, B, hkv = case["page"], _block(case["page"]), case["hkv"]
    plain = case["cache"] == "fp16"
    pools = [x.double() if plain else x.view(torch.float8_e4m3fn).double() for x in (s["kc"], s["vc"])]
    exps = None if s["scales"] is None else s["scales"].double() - 127.0
    table = s["table"].cpu()
    for b, (a, n, path) in enumerate(zip(_starts(case), _counts(case), _paths(case, seed))):
        def spot(place):
            return int(table[b, place // P]), place % P
        for i, pool in enumerate(pools):
            took = [pool[p, :, x].clone() if exps is None else pool[p, :, x] * torch.exp2(exps[p, :, x // B, i])[:, None]
                    for p, x in (spot(a + j) for j in path[:n])]
            if exps is None:
                for j in range(n):
                    p, x = spot(a + j)
                    pool[p, :, x] = took[j]
                continue
            for blk in sorted({(a + j) // B for j in range(n)}):
                mine = [j for j in range(n) if (a + j) // B == blk]
                if all(path[j] == j for j in mine):
                    continue
                p, x0 = spot(blk * B)
                big = torch.stack([took[j].abs().amax(-1) for j in mine]).amax(0)
                need = torch.ceil(torch.log2(big / 448.0)).clamp(K_MIN, K_MAX)
                if blk * B < a:
                    old = exps[p, :, x0 // B, i].clone()
                    need = torch.maximum(need, old)
                    pool[p, :, x0:x0 + a % B] *= torch.exp2(old - need)[:, None, None]
                for j in mine:
                    pool[p, :, spot(a + j)[1]] = took[j] * torch.exp2(-need)[:, None]
                exps[p, :, x0 // B, i] = need
    return tuple(pools) if exps is None else (pools[0], pools[1], torch.exp2(exps))


def exact(case: dict, seed: int):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "keep":
        return _exact_keep(case, seed)
    s = _inputs(case, seed)
    got = [_exact_kv(case, s, b, a, z) for b, (a, z) in enumerate(zip(_starts(case), _ends(case)))]
    return tuple(torch.cat([kv[j].transpose(0, 1) for kv in got]).contiguous() for j in (0, 1))
