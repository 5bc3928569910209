"""GPU tests of appends into pages whose offsets come near 32 bits."""

from __future__ import annotations

import pytest
import torch

import new_tokens as nt
import pa_amd
from helpers import D

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_device")]


@pytest.mark.parametrize("kind,P", [("fp16", 5_700_000), ("fp8", 11_300_000)])
def test_append_rope_in_a_page_of_gigabytes(kind, P):
    """A contiguous cache of one kv head as one page: rows for which there is no head reach 2^32 bytes and more past the
    page's first, and must not come round to it."""
    assert 2 ** 32 < 3 * P * D * (2 if kind == "fp16" else 1) and P * D * (2 if kind == "fp16" else 1) < 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(5)
    fill = 0x3C00 if kind == "fp16" else 0x38
    dt = torch.int16 if kind == "fp16" else torch.uint8
    pools = [torch.full((1, 1, P, D), fill, dtype=dt, device="cuda") for _ in range(2)]
    caches = [p.view(torch.float16) if kind == "fp16" else p for p in pools]
    n, start = 70, P - 100
    k, v, _ = (torch.empty((n, 3, 1, D), dtype=torch.float16, device="cuda").normal_(generator=g)[:, i] for i in range(3))
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
    rope = pa_amd.Rope(nt.freqs(128))
    for at in (start, 0):
        pa_amd.append_rope(None, k, v, *caches, dev([[0]]), dev([0, n]), dev([at]), rope)
    torch.cuda.synchronize()
    rows = torch.cat([torch.arange(start, start + n), torch.arange(n)]).cuda()
    got_v = pools[1][0, 0, rows]
    want = v[:, 0].contiguous().view(torch.int16) if kind == "fp16" else v[:, 0].to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(got_v, torch.cat([want, want]))
    assert bool((pools[0][0, 0, rows] != fill).any(-1).all())
    for p in pools:
        p[0, 0, rows] = fill
        assert int((p != fill).sum()) == 0   # no other row
