"""Every build of the 8-bit cache's kernels, by the sizes that choose it, against the formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

import test_cache_8bit_gpu as cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


# (query heads, key heads, head size): four rows a token, heads in each of the paddings to 64 values
FEW_HEADS = [(8, 2, 64), (8, 2, 48), (8, 2, 128), (8, 2, 96), (8, 2, 192), (8, 2, 176), (8, 2, 256), (8, 2, 208)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 4, 5, 8, 9, 12, 13, 16])
@pytest.mark.parametrize("nq,nkv,d", FEW_HEADS)
def test_few_rows_of_every_number_of_blocks(dtype, nq, nkv, d, tokens):
    """1 to 64 rows a request and key head; in one share, in shares, and in shares that the kernel cuts itself."""
    from paged_llm_rs_amd import kernels

    takes = kernels.library().pl_paged_attention_8bit_few(d, kernels.BF16 if dtype == torch.bfloat16 else kernels.F32)
    scene = cache.Scene([(tokens, 300), (1, 555), (tokens, tokens), (tokens, 640)], nq, nkv, d, 16, dtype)
    scene.check(scene.run())
    scene.check(scene.run(100), 100)
    if tokens * 4 > takes:
        return
    scene = cache.Scene([(tokens, 3000), (1, 5000), (tokens, 1700)], nq, nkv, d, 16, dtype)
    scene.check(scene.run())
    requests = [(tokens, 1100 + 300 * (s % 7)) for s in range(20)]
    scene = cache.Scene(requests, 32, 8, d, 16, dtype)
    scene.check(scene.run(max_ctx=60000))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 176, 192, 208, 256])
def test_many_rows_of_every_head_size(dtype, d):
    """Masked tiles in every build: prompts, portions, windows and blocks of positions, with key heads of 1 to 5 query heads."""
    for nq, nkv in ((4, 4), (8, 2), (5, 1)):
        scene = cache.Scene([(200, 200), (130, 700), (1, 90), (77, 77), (0, 3), (65, 1300)], nq, nkv, d, 16, dtype, extra_rows=1)
        for window in (0, 37, 300, -50):
            scene.check(scene.run(window, min_q_len=0), window)


@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (24, 12, 96), (64, 8, 128), (40, 20, 80)])
@pytest.mark.parametrize("requests,window", [
    ([(300, 300), (1500, 1500), (700, 700), (431, 431), (1001, 1001)], 0), ([(300, 300), (1500, 1500), (700, 700), (431, 431), (1001, 1001)], 333),
    ([(900, 2500), (1, 700), (640, 640), (3, 1100), (0, 5), (1, 1), (777, 1900)], 0), ([(900, 2500), (1, 700), (640, 640), (3, 1100), (0, 5), (1, 1), (777, 1900)], -500),
    ([(512, 4600)] + [(1, 700 + 250 * i) for i in range(15)], 0), ([(2100, 4600)] + [(1, 700 + 250 * i) for i in range(15)], 1000)])
def test_many_rows_with_eight_waves_a_workgroup(nq, nkv, d, requests, window):
    """Tiles that are widened for 256 rows: whole, in shares, under windows, beside short requests."""
    from paged_llm_rs_amd import kernels

    scene = cache.Scene(requests, nq, nkv, d, 16, torch.bfloat16, extra_rows=2)
    shares = kernels.shares_8bit(scene.n, len(requests), max(c for _, c in requests), nq, nkv, window, d, False)[3]
    assert kernels.library().pl_paged_attention_8bit_waves(scene.n, nq, nkv, d, shares, kernels.BF16) == 8
    if len(requests) == 16 and nq // nkv == 2 and window == 0:
        assert shares > 1
    scene.check(scene.run(window, min_q_len=0), window)
