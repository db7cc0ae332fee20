"""What the 8-bit cache's entry points refuse before anything is launched, and how many pages a byte budget holds (no GPU)."""

from __future__ import annotations

import pytest
import torch

from paged_llm_rs_amd import kernels
from paged_llm_rs_amd.cache import PagedCache
from paged_llm_rs_amd.cache.layout import CacheGroupLayout, CacheLayout, KVCacheSpec
from paged_llm_rs_amd.errors import ConfigError, TensorError


def layout(**more):
    return CacheLayout([CacheGroupLayout(KVCacheSpec(2, 64, **more), [0, 1]), CacheGroupLayout(KVCacheSpec(1, 32, window=64), [2])], {0: 0, 1: 0, 2: 1}, {})


def test_pages_of_a_byte_budget():
    lay = layout()
    assert lay.bytes_per_token(1) == 2 * (2 * 128 + 32) and lay.power_bytes == 2 * (2 * 2 + 1)
    per_page = 16 * lay.bytes_per_token(1) + lay.power_bytes
    assert lay.blocks_within(10 * per_page, 16, 1, lay.power_bytes) == 10 and lay.blocks_within(10 * per_page - 1, 16, 1, lay.power_bytes) == 9
    cache = PagedCache(lay, 16, 10, torch.bfloat16, "cpu", max_seqs=2, eight_bit=True)
    assert cache.bytes == 10 * per_page
    assert all(p.dtype == torch.float8_e4m3fn for p in cache.layer_pools(0))
    wide = PagedCache(lay, 16, 10, torch.bfloat16, "cpu", max_seqs=2)
    assert wide.bytes == 2 * 10 * 16 * lay.bytes_per_token(1) and wide.layer_pools(0)[0].dtype == torch.bfloat16
    with pytest.raises(ConfigError):
        PagedCache(layout(values_in_keys=True), 16, 10, torch.bfloat16, "cpu", eight_bit=True)


def test_the_c_entries_refuse_what_they_cannot_launch():
    lib = kernels.library()

    def refused(entry, good, **bad):
        for at, value in bad.values():
            args = list(good)
            args[at] = value
            assert entry(*args) == -1, (at, value)
            with pytest.raises(TensorError):
                kernels._check(-1)

    # q_len, ctx_len, S, table, width, block, free, num_free, rows, five results, stream
    refused(lib.pl_step_tables, [1, 1, 3, 1, 4, 16, 0, 0, 5, 1, 1, 1, 1, 1, 0], none=(2, 0), many=(2, 8193), width=(4, 0), block=(5, 0), free=(7, -1), rows=(8, -1))
    write = [1, 1, 512, 0, 0, 0, 1e-6, 0, 0, 0, 0, 0, 1, 1, 16, 64, 1, 1, 1, 1, 3, 4, 2, 64, 1, 0]
    refused(lib.pl_qk_norm_rope_kv_write_8bit, write, rot=(9, 65), odd=(9, 3), angles=(9, 64), block=(14, 0), rows=(15, 8), d=(23, 72), large=(23, 272), nkv=(22, 0), n=(20, -1))
    attend = [1, 256, 1, 1, 1, 1, 2, 3, 2, 1, 1, 4, 16, 64, 1, 1, 1, 1, 4, 2, 64, 0.1, 0, 512, 1, 512, 1, 0, 0, 1, 0]
    refused(lib.pl_paged_attention_8bit, attend, S=(6, 0), n=(7, 0), most=(8, 0), least=(9, 3), width=(11, 0), block=(12, 0), rows=(13, 8), nq=(18, 3), nkv=(19, 0), d=(20, 24), large=(20, 272),
            chunk=(23, 48), longest=(23, 4096), shares=(24, 0), no_room=(24, 2), many=(25, 32), many_shares=(26, 65536))


def test_the_shares_cover_every_context():
    """Whatever the sizes: the shares of a row block reach over every key that its rows may see, and a share is whole tiles."""
    for n in (1, 8, 64, 500, 8000):
        for requests in (1, 3, 64, 600):
            for max_ctx in (1, 31, 129, 4001, 30000, 1 << 20):
                for nq, nkv in ((1, 1), (16, 8), (64, 8), (12, 12)):
                    for window in (0, 1, 100, 5000, -64):
                        few, few_shares, many, many_shares = kernels.shares_8bit(n, requests, max_ctx, nq, nkv, window)
                        assert few % 32 == 0 and 32 <= few <= 2048 and many % 64 == 0 and many >= 64
                        for chunk, shares, tokens in ((few, few_shares, 64), (many, many_shares, 256)):
                            reach = max_ctx if window == 0 else min(max_ctx, abs(window) + tokens)
                            # a stretch of `reach` keys anywhere in the context touches at most so many shares
                            touched = min(-(-max_ctx // chunk), (reach - 1) // chunk + 2 if window else -(-max_ctx // chunk))
                            assert shares >= touched


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("d", [16, 96, 128, 256])
def test_the_shares_of_other_heads_cover_every_context(d, f32):
    for n, requests in ((1, 1), (64, 64), (527, 16), (4000, 5), (70000, 600)):
        for max_ctx in (1, 640, 641, 1500, 3100, 24000, 1 << 20):
            for nq, nkv in ((16, 8), (64, 8), (8, 1), (300, 100)):
                for window in (0, 100, -3000):
                    few, few_shares, many, many_shares = kernels.shares_8bit(n, requests, max_ctx, nq, nkv, window, d, f32)
                    assert few % 32 == 0 and 32 <= few <= 2048 and many % 64 == 0 and many >= 64
                    for chunk, shares, tokens in ((few, few_shares, 64), (many, many_shares, 256)):
                        reach = max_ctx if window == 0 else min(max_ctx, abs(window) + tokens)
                        assert shares >= min(-(-max_ctx // chunk), (reach - 1) // chunk + 2 if window else -(-max_ctx // chunk))
