"""Attention over 8-bit pages that hold values which are not finite: a row is what the keys that it sees make it, whatever stands at the others."""

from __future__ import annotations

import pytest
import torch

import test_cache_8bit_gpu as cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


def seen_by(scene, s, window):
    """[tokens, keys]: which keys the tokens of request s see."""
    q, c = scene.requests[s]
    pos, key = torch.arange(c - q, c, device=cache.DEV).view(-1, 1), torch.arange(c, device=cache.DEV).view(1, -1)
    seen = key <= pos
    if window > 0:
        seen &= key > pos - window
    if window < 0:
        seen &= key >= pos - pos % -window
    return seen


def spoil(scene, s, position, head, columns, which=1):
    """NaN (the byte that a value which is not finite is kept as) into columns of a key's row."""
    page = int(scene.table[s, position // scene.block])
    pool = scene.pages.pools[which].view(torch.uint8).view(-1, scene.nkv, scene.d)
    pool[page * scene.block + position % scene.block, head, columns] = 0x7f if position % 2 else 0xff


LAYOUTS = [(16, 8, 128), (8, 2, 64), (6, 2, 80), (4, 4, 32), (8, 1, 192), (8, 4, 256), (12, 12, 96)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", LAYOUTS)
@pytest.mark.parametrize("requests", [[(8, 40), (4, 700), (5, 1100), (2, 33)], [(200, 200), (130, 700), (1, 90), (9, 1100), (65, 1300)]])
def test_a_nan_value_reaches_the_tokens_that_see_it_alone(dtype, nq, nkv, d, requests):
    """The last tokens' values, those in front of a window, of one column, of all: the others are what the keys that they see make them, to the same tolerance as without."""
    group = nq // nkv
    for window in (0, 20, -24):
        scene = cache.Scene(requests, nq, nkv, d, 16, dtype)
        clean = scene.run(window, min_q_len=1)
        scene.check(clean, window)
        spoilt = []
        for s, (q, c) in enumerate(requests):
            for position, head, columns in ((c - 1, 0, slice(None)), (c - 1 - q // 2, nkv - 1, slice(3, 4)), (max(c - q - 1, 0), nkv - 1, slice(d - 1, d)), (max(c - q - 9, 0), 0, slice(5, 9)),
                                            (max(c - q // 3 - 1, 0), nkv // 2, slice(d // 2, None))):
                spoil(scene, s, position, head, columns)
                spoilt.append((s, position, head, columns))
        out = scene.run(window, min_q_len=1)
        bad = torch.zeros(scene.n, nkv, group, d, dtype=torch.bool, device=cache.DEV)
        for s, position, head, columns in spoilt:
            at, q = scene.starts[s], requests[s][0]
            rows = torch.zeros(scene.n, dtype=torch.bool, device=cache.DEV)
            rows[at:at + q] = seen_by(scene, s, window)[:, position]
            where = torch.zeros(d, dtype=torch.bool, device=cache.DEV)
            where[columns] = True
            bad[:, head] |= rows.view(-1, 1, 1) & where
        bad = bad.view(scene.n, nq * d)
        assert bool(out[bad].isnan().all())
        out[bad] = clean[bad]
        scene.check(out, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (6, 2, 80)])
def test_a_nan_key_reaches_the_tokens_that_see_it_alone(dtype, nq, nkv, d):
    requests = [(8, 40), (150, 300), (4, 1100)]
    for window in (0, 20):
        scene = cache.Scene(requests, nq, nkv, d, 16, dtype)
        clean = scene.run(window)
        bad = torch.zeros(scene.n, nkv, nq // nkv, d, dtype=torch.bool, device=cache.DEV)
        for s, (q, c) in enumerate(requests):
            for position in (c - 1, c - 1 - q // 2):
                spoil(scene, s, position, 1, slice(2, 3), which=0)
                bad[scene.starts[s]:scene.starts[s] + q, 1] |= seen_by(scene, s, window)[:, position].view(-1, 1, 1)
        bad = bad.view(scene.n, nq * d)
        out = scene.run(window)
        assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_past_the_largest_bfloat16(dtype):
    """A page whose power makes its largest values infinite in bfloat16: the tokens that see such a key have nothing finite there, those in front of it their own values."""
    scene = cache.Scene([(40, 40), (6, 30)], 4, 2, 64, 16, dtype)
    for s, position in ((0, 38), (1, 29)):
        page = int(scene.table[s, position // 16])
        scene.pages.powers[1].view(torch.uint8)[page, 1] = 127 + 120
        pool = scene.pages.pools[1].view(torch.uint8).view(-1, 2, 64)
        pool[page * 16:page * 16 + 16, 1] = 0                       # (values of the page are nothing but ...)
        pool[page * 16 + position % 16, 1, 7] = 0x7e                # 448
        pool[page * 16 + position % 16, 1, 9] = 0xfe                # -448
    scene.q.mul_(0.1)
    out = scene.run().view(scene.n, 2, 2, 64)
    for s, (q, c) in enumerate(scene.requests):
        position = 38 if s == 0 else 29
        rows = out[scene.starts[s]:scene.starts[s] + q]
        late = c - q + torch.arange(q, device=cache.DEV) >= position
        assert not bool(rows[late][:, 1, :, [7, 9]].isfinite().any())
        assert bool(rows[~late].isfinite().all()) and bool(rows[late][:, 1, :, 10:].isfinite().all()) and bool(rows[late][:, 0].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,max_ctx", [([(150, 400), (5, 3000), (3, 900), (1, 50)], 3000), ([(2 + s % 4, 1500 + 97 * s) for s in range(40)], 60000), ([(700, 2500), (300, 300)], 2500)])
def test_a_nan_value_among_shares(dtype, requests, max_ctx):
    """Few rows beside many, whose shares stand in other places of the room; contexts that the kernel cuts itself; many rows in shares: NaN at the last tokens, before them, and far in front (which all rows see)."""
    scene = cache.Scene(requests, 32, 8, 64, 16, dtype)
    for window in (0, 70):
        clean = scene.run(window, max_ctx=max_ctx)
        scene.check(clean, window)
        held = scene.pages.clone()
        bad = torch.zeros(scene.n, 8, 4, 64, dtype=torch.bool, device=cache.DEV)
        for s, (q, c) in enumerate(requests):
            for position, head, columns in ((c - 1, 1, slice(None)), (c - 1 - q // 2, 2, slice(0, 5)), (max(c - q - 20, 0), 3, slice(7, 8)), (c // 5, 4, slice(None)), (c // 5, 5, slice(9, 10)), (c - 1, 5, slice(8, 12)),
                                            (c - 1 - q // 3, 5, slice(40, 50))):
                spoil(scene, s, position, head, columns)
                bad[scene.starts[s]:scene.starts[s] + q, head, :, columns] |= seen_by(scene, s, window)[:, position].view(-1, 1, 1)
        bad = bad.view(scene.n, -1)
        out = scene.run(window, max_ctx=max_ctx)
        assert bool(out[bad].isnan().all())
        out[bad] = clean[bad]
        scene.check(out, window)
        scene.pages = held
