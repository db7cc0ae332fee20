"""That the 8-bit attention has shares enough for every block of rows, counted row by row from what its tokens see (no GPU)."""

from __future__ import annotations

import random

import pytest

from paged_llm_rs_amd import kernels


def first_seen(position, window):
    """The first key that the token at a position sees."""
    if window > 0:
        return max(position - window + 1, 0)
    if window < 0:
        return position // -window * -window
    return 0


def touched(first_token, last_token, window, chunk):
    """Shares, which begin at whole ones, that hold a key which some of the tokens see: the first token sees the earliest, the last the latest."""
    seen = [first_seen(first_token, window), last_token]
    return seen[1] // chunk - seen[0] // chunk + 1


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 256])
def test_every_block_of_rows_has_its_shares(d, f32):
    draw = random.Random(1000 * d + f32)
    takes = kernels.library().pl_paged_attention_8bit_few(d, kernels.F32 if f32 else kernels.BF16)
    cut = 0
    for _ in range(4000):
        nkv = draw.choice([1, 2, 3, 8, 12])
        group = draw.choice([1, 2, 3, 4, 5, 8, 40, 100])
        window = draw.choice([0, 0, 1, 3, 100, 1000, 5000, -1, -7, -64, -1000, -4096])
        max_ctx = int(2 ** draw.uniform(0, 17))
        requests = draw.choice([1, 1, 2, 8, 64, 65, 300])
        ctx = draw.choice([max_ctx, draw.randint(1, max_ctx)])
        brings = draw.choice([1, min(ctx, draw.randint(1, 70)), draw.randint(1, ctx)])
        n = brings + requests - 1
        few, few_shares, many, many_shares = kernels.shares_8bit(n, requests, max_ctx, nkv * group, nkv, window, d, f32)
        assert few % 32 == 0 and 32 <= few <= 2048 and many % 64 == 0 and many >= 64
        rows = brings * group
        # all rows of a request together, by tokens or (where the kernel cuts a request's keys itself) by how many keys they are
        if rows <= takes:
            assert few_shares >= touched(ctx - brings, ctx - 1, window, few)
            assert few * few_shares >= ctx - first_seen(ctx - brings, window)
        # blocks of 128 rows and of 256
        if rows > 16:
            for block in (128, 256):
                for begin in {0, (rows - 1) // block * block, draw.randint(0, (rows - 1) // block) * block}:
                    end = min(begin + block, rows) - 1
                    assert many_shares >= touched(ctx - brings + begin // group, ctx - brings + end // group, window, many), (n, requests, max_ctx, nkv, group, window)
        cut += few_shares > 1 and many_shares > 1
    assert cut > 200          # (draws in which both kernels cut their keys)
