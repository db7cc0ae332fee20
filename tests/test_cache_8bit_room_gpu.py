"""What room a call of the 8-bit attention takes on the card, and that the kernels keep to it."""

from __future__ import annotations

import pytest
import torch

import test_cache_8bit_gpu as cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


def taken(call):
    """Bytes that a call had beside what was there, at most."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_fresh_prompt_takes_no_room(dtype):
    scene = cache.Scene([(5000, 5000)], 16, 8, 64, 16, dtype)
    out = torch.empty(scene.n, 16 * 64, dtype=dtype, device="cuda:0")
    assert taken(lambda: scene.run(out=out)) <= 1 << 20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (6, 2, 80), (8, 1, 64)])
def test_single_tokens_beside_a_portion_have_room_for_themselves(dtype, nq, nkv, d):
    """Few rows are numbered by request and key head, many by the step's rows: both put together, and both beside padding and a request of no rows."""
    from paged_llm_rs_amd import kernels

    requests = [(1, 3000), (300, 4100), (1, 17), (0, 9), (2, 2500), (3, 2), (16, 1500), (1, 1), (40, 3500)]
    scene = cache.Scene(requests, nq, nkv, d, 16, dtype, extra_rows=3)
    _, few, _, many, places = kernels._plan_8bit(scene.n, len(requests), 300, 0, 4100, nq, nkv, 0, d, kernels._code(scene.q, "q"))
    assert few > 1 and places == len(requests) * nkv * 16 * few + (scene.n * nq * many if many > 1 else 0) < scene.n * nq * max(few, many) * 2
    out = torch.full((scene.n, nq * d), -7.0, dtype=dtype, device="cuda:0")
    assert taken(lambda: scene.run(min_q_len=0, out=out)) <= 4 * places * (d + 2) + (1 << 20)
    scene.check(out)
    scene.check(scene.run(700, min_q_len=0), 700)
