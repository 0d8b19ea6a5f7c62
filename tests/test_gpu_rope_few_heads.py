"""Rotary positions of few heads and many tokens, which a work-group takes several of: against 64 bits with the
tolerance of test_gpu_rope.py."""

import pytest
import torch

from ananta_ocr_amd import rope
from test_gpu_rope import DEV, TYPES, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T, H, Hkv, D, m, start", [(1023, 1, 1, 64, 32, 0), (1024, 1, 1, 64, 32, 0), (1501, 1, 1, 128, 64, 0),
                                                    (2047, 2, 1, 64, 16, 32), (1030, 1, 1, 20, 5, 4), (1030, 3, 0, 64, 32, 0)])
def test_append_of_many_tokens(T, H, Hkv, D, m, start, dtype, interleaved):
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV)
    q, k, v = x.split((H, Hkv, Hkv), 1)
    page, pages = 16, (T + 15) // 16 + 2
    kc, vc = (torch.randn(pages, page, Hkv, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    pos = torch.randint(0, 10 ** 5, (T,), generator=g).to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[::7] = -1
    slots = slots.to(DEV)
    f, _ = rope.inv_freq(2 * m, device=DEV)
    want_k, want_v = kc.clone(), vc.clone()
    out = rope.rope_append(q, k, v, pos, slots, kc, vc, f, interleaved=interleaved, start=start)
    _close(out, q, pos, f, interleaved, start)
    if not Hkv:
        return
    k2 = rope.apply_rope(k, None, pos, f, interleaved=interleaved, start=start)
    _close(k2, k, pos, f, interleaved, start)
    live = slots >= 0
    want_k.view(-1, Hkv, D)[slots[live]] = k2[live]
    want_v.view(-1, Hkv, D)[slots[live]] = v[live]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.parametrize("interleaved", [False, True])
def test_batches_that_end_inside_a_work_group(interleaved):
    """Four tokens a work-group, of two batch rows with positions and strides of their own."""
    g = torch.Generator().manual_seed(1)
    f, _ = rope.inv_freq(64, device=DEV)
    x = torch.randn(3, 2, 401, 64, generator=g).to(DEV).transpose(1, 2)
    pos = torch.randint(0, 9000, (3, 802), generator=g).to(DEV)[:, ::2]
    _close(rope.apply_rope(x, None, pos, f, interleaved), x, pos, f, interleaved)
