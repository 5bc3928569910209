"""Outputs of the new-token operators that share memory with other rows of the call are refused, and rows that only lie
between each other are not (CPU: the refusals come before anything is launched; what is taken runs on the GPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import new_tokens as nt
import pa_amd
from helpers import D
from pa_amd import _lib

BAD = _lib.PA_ERR_INVALID_ARGUMENT
A = 1 << 24   # an address that nothing reads: every call on the CPU is refused first
H = 2 * D     # bytes of a head


def rows(at, heads, stride, out=None, out_stride=None):
    r = _lib.HeadRows()
    r.in_, r.heads, r.in_stride, r.eps = at, heads, stride, 1e-6
    r.out, r.out_stride = out, stride if out_stride is None else out_stride
    return r


def norm(q, k, n):
    ref = lambda r: None if r is None else ctypes.byref(r)   # noqa: E731
    return _lib.load().pa_norm_rope(None, ref(q), ref(k), None, n, None)


def append(q, k, v, v_stride, n):
    a = _lib.AppendArgs()
    far = 1 << 40
    a.num_tokens, a.num_entries, a.tok_begin, a.start_pos = n, 1, far, far
    a.v, a.v_stride, a.k_cache, a.v_cache = v, v_stride, far, far
    a.block_table, a.block_table_stride, a.num_table_rows, a.num_pages = far, 4, 2, 8
    a.page_size, a.k_scale, a.v_scale = 16, 1.0, 1.0
    return _lib.load().pa_append_rope(0, ctypes.byref(a), None, ctypes.byref(q), ctypes.byref(k), None)


def message() -> str:
    return _lib.load().pa_last_error().decode()


# A buffer of 8 columns of heads, q in the first two, k in the next, v behind it.
S = 8 * D
FREE = 1 << 30


@pytest.mark.parametrize("n", [1, 2, 100])
@pytest.mark.parametrize("q_out,k_out,word", [
    (A + 2 * H, FREE, "q's output overlaps k"), (A + H, FREE, "the output overlaps the rows"),
    (FREE, A + H, "k's output overlaps q"), (FREE, FREE, "the outputs overlap"), (FREE, FREE + H, "the outputs overlap"),
    (A, A, "the outputs overlap"), (A + 2 * H, A, "overlaps"),
])
def test_norm_rope_refuses_outputs(n, q_out, k_out, word):
    assert norm(rows(A, 2, S, q_out), rows(A + 2 * H, 1, S, k_out), n) == BAD and word in message(), message()


@pytest.mark.parametrize("out,stride,n", [
    (A + 2 * S - H, S, 3),        # ends in the next token's row
    (A + 2 * S * 4, S, 5),        # starts at the last token's row
    (A - 2 * S * 4, S, 5),        # its last row at the first token's
    (A + 3 * H, 2 * D, 100),      # between them, with another stride
    (A, 4 * D, 5),                # the rows' start with another stride
    (A - 4 * H, 5 * D, 2),        # its second row is one head into the first token's (from A - 3 * H on: behind it)
])
def test_norm_rope_refuses_rows_among_each_other(out, stride, n):
    assert norm(rows(A, 2, S, out, stride), None, n) == BAD and "overlaps" in message()


def test_append_rope_refuses_outputs():
    for n in (1, 7):
        for out, word in ((A + 2 * H, "overlaps k"), (A + 3 * H, "overlaps v"), (A + H, "overlaps the rows")):
            assert append(rows(A, 2, S, out), rows(A + 2 * H, 1, S), A + 3 * H, S, n) == BAD and word in message(), message()


def test_any_rows_against_every_byte():
    """Whether rows share a byte, against all of them listed. (What is not refused goes on to the launch, which finds no
    device here: never on a machine that has one.)"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the calls that are taken would run")
    rng = np.random.default_rng(0)
    seen = [0, 0]
    for _ in range(4000):
        n, heads = int(rng.integers(1, 7)), int(rng.integers(1, 4))
        step = heads * D + 8 * int(rng.integers(0, 60)) if rng.random() < 0.8 else 8 * int(rng.integers(0, 100))
        out_step = step if rng.random() < 0.6 else heads * D + 8 * int(rng.integers(0, 60))
        if n > 1 and out_step < heads * D:
            continue
        out = A + 16 * int(rng.integers(-n * step // 8 - 60, n * step // 8 + 60))
        if out == A and (n == 1 or step == out_step):
            continue
        lists = [set().union(*(range(at + 2 * i * s, at + 2 * i * s + heads * H, 16) for i in range(n)))
                 for at, s in ((A, step), (out, out_step))]
        meets = bool(lists[0] & lists[1])
        seen[meets] += 1
        assert norm(rows(A, heads, step, out, out_step), None, n) == (BAD if meets else _lib.PA_ERR_DEVICE)
    assert min(seen) > 500


@pytest.mark.gpu
@pytest.mark.usefixtures("gpu_device")
def test_rows_between_each_other_are_taken():
    """Outputs in other columns of their inputs' buffer, of one stride and of another, and outputs that are q and k
    in place: the values of calls with outputs of their own, and nothing else of the buffer changes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    n, hq, hkv = 21, 3, 2
    rope = pa_amd.Rope(nt.freqs(128))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    buf = torch.empty((n, 2 * (hq + hkv) + 1, D), dtype=torch.float16, device="cuda").normal_(generator=g)
    q, k = buf[:, :hq], buf[:, hq:hq + hkv]
    want = [t.clone() for t in pa_amd.norm_rope(q, k, pos, rope)]
    before = buf.clone()
    qo, ko = buf[:, hq + hkv:2 * hq + hkv], buf[:, 2 * hq + hkv:2 * (hq + hkv)]
    pa_amd.norm_rope(q, k, pos, rope, q_out=qo, k_out=ko)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    assert torch.equal(buf[:, :hq + hkv], before[:, :hq + hkv]) and torch.equal(buf[:, -1], before[:, -1])
    pa_amd.norm_rope(q, k, pos, rope, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # Rows 4 heads apart, outputs in the gaps 8 heads apart.
    flat = torch.empty((8 * n, D), dtype=torch.float16, device="cuda").normal_(generator=g)
    x, out = flat[:4 * n].view(n, 4, D)[:, :1], flat.view(n, 8, D)[:, 2:3]
    want, _ = pa_amd.norm_rope(x, None, pos, rope)
    kept = x.clone()
    pa_amd.norm_rope(x, None, pos, rope, q_out=out)
    assert torch.equal(out, want) and torch.equal(x, kept)
