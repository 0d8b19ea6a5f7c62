"""Page calls (kv_pages) at sizes past one grid."""

import pytest
import torch

from ananta_ocr_amd import kv_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_more_pairs_and_caches_than_a_grid_has():
    """A pool of a million one-token pages in 36 caches: half of its pages are pairs of the copy, more
    than a launch's grid has of them, and with the caches more work-groups than it could have."""
    n, used = (1 << 20) + 3, 300001
    g = torch.Generator().manual_seed(2)
    live = torch.randperm(n, generator=g)[:used].to(torch.int32)
    caches = [torch.randint(0, 256, (n, 1), generator=g, dtype=torch.uint8).to(DEV) for _ in range(36)]
    refs = torch.zeros(n, dtype=torch.int32)
    refs[live.long()] = 1
    refs, table, lens = refs.to(DEV), live[None].to(DEV), _i32([used])
    want = [c[table[0].long()] for c in caches]
    refs2, table2, frm, to = kv_pages.compact_pages(refs, table, lens, 1)
    assert int((frm >= 0).sum()) > 65535 and frm.numel() == n // 2
    kv_pages.copy_pages(kv_pages.PageCaches(caches), frm, to)
    assert torch.equal(table2[0].sort().values, torch.arange(used, dtype=torch.int32, device=DEV))
    assert torch.equal(refs2, (torch.arange(n, device=DEV) < used).to(torch.int32))
    for c, w in zip(caches, want):
        assert torch.equal(c[table2[0].long()], w)
