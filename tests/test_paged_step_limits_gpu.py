"""fr_paged_step at the largest sizes it accepts, max_tokens or num_pages
2^30 - 1: sums past them refuse the step and change nothing, one that fits
exactly is taken."""
from __future__ import annotations

import pytest
import torch

from forgert_b200 import _lib
from forgert_b200 import attention as A

pytestmark = pytest.mark.gpu

MOST = (1 << 30) - 1
I32 = dict(dtype=torch.int32, device="cuda")


def step(kv, new, width, page_size, num_pages, max_tokens):
    B = len(new)
    a = dict(kv=torch.tensor(kv, **I32), new=torch.tensor(new, **I32), table=torch.full((B, width), -1, **I32),
             stack=torch.arange(num_pages, **I32), count=torch.tensor([num_pages], **I32),
             offsets=torch.full((B + 1,), -7, **I32), positions=torch.full((max_tokens,), -7, **I32),
             slots=torch.full((max_tokens,), -7, dtype=torch.int64, device="cuda"), status=torch.full((1,), -7, **I32))
    A.paged_step(a["kv"], a["new"], a["table"], a["stack"], a["count"], a["kv"], a["count"], a["offsets"], a["positions"],
                 a["slots"], a["status"], B, page_size, num_pages, width, max_tokens)
    torch.cuda.synchronize()
    return a


def refused(a, kv, num_pages):
    assert a["kv"].tolist() == kv and int(a["count"]) == num_pages
    assert int(a["table"].max()) == -1 and torch.equal(a["stack"], torch.arange(num_pages, **I32))
    assert int(a["offsets"].abs().max()) == 0 and int(a["positions"].abs().max()) == 0
    assert int(a["slots"].max()) == -1 and int(a["slots"].min()) == -1


def test_tokens_past_the_largest_limit():
    """Two warps' sums of 2^30 each."""
    a = step([0] * 64, [1 << 25] * 64, 1 << 10, 1 << 15, 64, MOST)
    assert int(a["status"]) == _lib.FR_STEP_TOO_MANY
    refused(a, [0] * 64, 64)


def test_pages_past_the_largest_pool():
    """Requests that claim to hold 2^31 pages of a pool of 2^30 - 1 end."""
    kv = [1 << 25] * 64
    a = step(kv, [-1] * 64, 1 << 25, 1, MOST, 64)
    assert int(a["status"]) == _lib.FR_STEP_BAD_FREE
    refused(a, kv, MOST)


def test_tokens_that_fit_exactly():
    n, page, pages = 1 << 24, 1 << 15, 1 << 15
    new = [n] * 63 + [n - 1]
    a = step([0] * 64, new, 1 << 10, page, pages, MOST)
    assert int(a["status"]) == _lib.FR_STEP_OK
    assert a["kv"].tolist() == new and int(a["count"]) == 0
    assert a["offsets"].tolist() == [b * n for b in range(64)] + [MOST]
    per = n // page
    pos = torch.arange(n, dtype=torch.int64, device="cuda")
    for b in range(64):
        at = slice(b * n, b * n + new[b])
        p = pos[:new[b]]
        ids = pages - 1 - (b * per + p // page)                 # popped in (request, block) order
        assert torch.equal(a["positions"][at].long(), p)
        assert torch.equal(a["slots"][at], ids * page + p % page)
