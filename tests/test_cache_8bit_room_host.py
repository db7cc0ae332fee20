"""How much room the 8-bit attention asks for what its shares leave, from its rules alone (no GPU)."""

from __future__ import annotations

import pytest

from paged_llm_rs_amd import kernels

MB = 2 ** 20


def room(n, requests, most, least, max_ctx, nq, nkv, d=128, f32=False, window=0):
    """Bytes, as ``paged_attention_8bit`` asks for them."""
    plan = kernels._plan_8bit(n, requests, most, least, max_ctx, nq, nkv, window, d, kernels.F32 if f32 else kernels.BF16)
    assert plan[:4] == kernels.shares_8bit(n, requests, max_ctx, nq, nkv, window, d, f32)
    return 4 * plan[4] * (d + 2)


@pytest.mark.parametrize("d,f32", [(128, False), (64, False), (256, True), (16, True)])
@pytest.mark.parametrize("nq,nkv", [(16, 8), (32, 8), (64, 8), (12, 12), (8, 1)])
def test_fresh_prompts_take_next_to_none(nq, nkv, d, f32):
    """Only the kernel of many rows runs: its shares times its rows are at most what the chip works on at a time, 256 workgroups of 256 rows, and those cut in two."""
    for tokens in (100, 700, 8100, 32768, 131072):
        for requests in (1, 2, 7):
            assert room(tokens * requests, requests, tokens, tokens, tokens, nq, nkv, d, f32) <= 2 * 256 * 256 * (d + 2) * 4


def test_portions_beside_single_tokens_at_long_contexts():
    """The few rows have 16 rows a request and key head, the many ones as above."""
    for n, requests, max_ctx, nq, nkv in ((2048, 16, 131072, 64, 8), (527, 16, 4600, 16, 8), (8192, 9, 49152, 32, 8), (512, 2, 1000000, 64, 8), (2048, 65, 131072, 32, 8)):
        shares = kernels.shares_8bit(n, requests, max_ctx, nq, nkv)
        many = 2 * 256 * 256 * 130 * 4
        assert room(n, requests, n - requests + 1, 1, max_ctx, nq, nkv) <= requests * nkv * 16 * shares[1] * 130 * 4 + many
        assert room(n, requests, n - requests + 1, 1, max_ctx, nq, nkv) <= 300 * MB
        # a portion on its own, padded or not
        assert room(n, 2, n, 16, max_ctx, nq, nkv) <= many


def test_few_rows_have_room_for_their_own():
    for nq, nkv, each in ((16, 8, 1), (32, 8, 1), (64, 8, 5), (12, 12, 9), (8, 1, 3)):
        for requests in (1, 8, 64, 200):
            n = requests * each
            few, shares, _, _ = kernels.shares_8bit(n, requests, 24000, nq, nkv)
            assert room(n, requests, each, each, 24000, nq, nkv) <= (n * nq * shares * 130 * 4 if shares > 1 else 0)
    # one draft of eight among single tokens
    assert room(71, 64, 8, 1, 24000, 32, 8) <= 71 * 32 * kernels.shares_8bit(71, 64, 24000, 32, 8)[1] * 130 * 4
    # contexts in one share need none
    assert room(64, 64, 1, 1, 600, 16, 8) == 0 and room(2000, 1, 2000, 2000, 2000, 16, 8) == room(2000, 1, 2000, 2000, 2000, 16, 8)


def test_no_room_is_refused():
    lib = kernels.library()
    # the kernel of many rows alone, whole: no room needed however many shares few rows would have (refused for its head size, behind which nothing is launched)
    assert lib.pl_paged_attention_8bit_places(1, 8100, 8100, 8100, 32, 8, 128, 32, 1, kernels.BF16) == 0
    assert lib.pl_paged_attention_8bit_places(1, 8100, 8100, 8100, 32, 8, 128, 32, 3, kernels.BF16) == 3 * 8100 * 32
    assert lib.pl_paged_attention_8bit_places(16, 527, 512, 1, 16, 8, 128, 3, 7, kernels.BF16) == 16 * 8 * 16 * 3 + 7 * 527 * 16
    attend = [1, 512, 1, 1, 1, 1, 2, 100, 99, 1, 1, 4, 16, 64, 1, 1, 1, 1, 4, 2, 64, 0.1, 0, 512, 1, 512, 1, 0, 0, 1, 0]
    for at in (24, 26):
        args = list(attend)
        args[at] = 2
        assert lib.pl_paged_attention_8bit(*args) == -1
        assert b"room" in lib.pl_last_error()
