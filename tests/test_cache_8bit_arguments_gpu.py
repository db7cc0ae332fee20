"""Arguments of the 8-bit cache's operators that do not fit the kernels' 32 bits, or are not there."""

from __future__ import annotations

import sys

import pytest
import torch

import test_cache_8bit_gpu as cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 33 + 5, sys.maxsize, -2 ** 31, -2 ** 33 - 5])
def test_a_window_past_32_bits_hides_nothing(window):
    scene = cache.Scene([(1, 300), (3, 40), (70, 200)], 4, 2, 64, 16, torch.bfloat16)
    scene.check(scene.run(window))


def test_sizes_and_scales_past_32_bits_are_refused():
    from paged_llm_rs_amd import kernels
    from paged_llm_rs_amd.errors import TensorError

    scene = cache.Scene([(1, 300), (3, 40)], 4, 2, 64, 16, torch.bfloat16)
    for max_ctx in (2 ** 31, 2 ** 32 + 64, 2 ** 40):
        with pytest.raises(TensorError):
            scene.run(max_ctx=max_ctx)
    for scale in (1e39, 1e-46, 3.3e38):
        scene.scale = scale
        with pytest.raises(TensorError):
            scene.run()
    for other in (dict(rows=2 ** 32 + 4), dict(block_size=2 ** 32 + 16), dict(block_size=2 ** 31)):
        a = dict(q_len=scene.q_len, ctx_len=scene.ctx_len, block_table=scene.table, block_size=16, free_pages=None, rows=4)
        a.update(other)
        with pytest.raises(TensorError):
            kernels.step_tables(**a)


def test_missing_tables_and_slots_are_refused():
    from paged_llm_rs_amd.errors import TensorError

    pages = cache.Pages(2, 16, 2, 64)
    rows = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=cache.DEV)
    angles = torch.zeros(30, 32, device=cache.DEV)
    at = cache.i32([0, 1, 2])
    for other in (dict(cos=None, sin=angles, rot=64), dict(cos=angles, sin=None, rot=64), dict(slots=None)):
        a = dict(slots=at, positions=at, nq=4)
        a.update(other)
        with pytest.raises(TensorError):
            cache.write(pages, rows, **a)
