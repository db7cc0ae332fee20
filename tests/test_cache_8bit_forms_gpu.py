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


# ---- the write of many rows ----------------------------------------------------------------------------------------------

def least_power(top):
    """The bytes of the least powers of two whose 448-fold holds ``top`` (64-bit, not negative)."""
    part, exponent = torch.frexp(top)
    return torch.where(top > 0, exponent - 9 + (part > 0.875).int(), torch.full_like(exponent, -126)).clamp(min=-126) + 127


def plain_write(pages, which, rows, slots, slack):
    """What the pools ought to hold and the least and largest power of every page and head: ``rows`` [n, nkv, d] in 64 bits, ``slots`` a list (-1: nowhere), values known to within
    ``slack`` of themselves.  (values in 64 bits before their rounding, which slots they are in, least power, largest power, pages written)"""
    block = pages.block
    live = torch.tensor([r for r, s in enumerate(slots) if s >= 0], device=rows.device)
    at = torch.tensor([s for s in slots if s >= 0], device=rows.device)
    page = at // block
    # a page is begun anew where its first slot is among those written
    first = torch.full((pages.powers[which].shape[0],), block, device=rows.device, dtype=torch.long).scatter_reduce_(0, page, at % block, "amin")
    top = torch.zeros(pages.powers[which].shape, dtype=torch.float64, device=rows.device).index_reduce_(0, page, rows[live].abs().amax(-1), "amax")
    had = torch.where(((first > 0) & (first < block)).view(-1, 1), pages.powers[which].view(torch.uint8).int(), torch.zeros_like(pages.powers[which].view(torch.uint8).int()))
    return at, live, page, first, torch.maximum(least_power(top * (1 - slack)), had), torch.maximum(least_power(top * (1 + slack)), had)


def check_write(pages, before, which, rows, slots, exact):
    """``exact``: the values took no arithmetic on the way, so powers and bytes are those of the definition.  Else they are off by at most 1e-5 of the row's largest before the rounding (32-bit norms
    and rotations), so a maximum near a border may fall on either side, and a byte is off by half a step of e4m3 beside that."""
    block, nkv, d = pages.block, pages.nkv, pages.d
    at, live, page, first, least, most = plain_write(before, which, rows, slots, 0.0 if exact else 1e-5)
    got, was = (p.powers[which].view(torch.uint8).int() for p in (pages, before))
    written = first < block
    assert torch.equal(got[~written], was[~written])
    assert bool(((got >= least) & (got <= most))[written].all())
    unit = torch.exp2(got.double() - 127)
    held, then = (p.pools[which].double().view(-1, nkv, d) for p in (pages, before))
    want = rows[live]
    u = unit[page].unsqueeze(-1)
    if exact:
        assert torch.equal(pages.pools[which].view(-1, nkv, d)[at].view(torch.uint8), (want / u).float().to(cache.E4M3).view(torch.uint8))
    off = (held[at] * u - want).abs()
    assert bool((off <= torch.maximum(cache.HALF_E4M3 * want.abs(), 2.0 ** -10 * u) + (0 if exact else 1e-5) * want.abs().amax(-1, keepdim=True)).all())
    # what was there in front of a page's new rows: as it was, or rounded again in the new unit, to the bit
    place = torch.arange(held.shape[0], device=held.device)
    kept = written[place // block] & (place % block < first[place // block])
    # (nearest, ties to even, of what a power of two divides exactly)
    fewer = torch.exp2((was - got).double())[place // block].unsqueeze(-1)
    assert torch.equal(pages.pools[which].view(-1, nkv, d)[kept].view(torch.uint8), (then * fewer)[kept].float().to(cache.E4M3).view(torch.uint8))
    touched = torch.zeros(held.shape[0], dtype=torch.bool, device=held.device)
    touched[at] = True
    same = ~(touched | kept)
    assert torch.equal(pages.pools[which].view(torch.uint8)[same], before.pools[which].view(torch.uint8)[same])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d,block,rot,normed,neighbours,waves", [
    (16, 8, 128, 16, 128, True, False, 4), (16, 8, 128, 5, 128, True, False, 4), (16, 8, 128, 3, 128, True, False, 1), (8, 8, 128, 128, 64, False, False, 4), (4, 8, 64, 16, 64, True, False, 4),
    (4, 8, 64, 8, 30, True, False, 1), (4, 8, 96, 300, 90, True, False, 4), (8, 8, 256, 16, 256, True, False, 4), (8, 8, 256, 2, 0, True, False, 1), (12, 12, 32, 32, 32, False, True, 4),
    (0, 12, 16, 16, 0, False, False, 1), (8, 8, 176, 1, 22, True, True, 1)])
def test_many_rows_into_their_pages(dtype, nq, nkv, d, block, rot, normed, neighbours, waves):
    """Steps of enough rows to be looked through 32 at a time, a wave or four to a run: prompts that end inside such a tile, requests that begin inside a page whose power grows or does not, runs that
    cross tiles, several runs a tile, rows of padding between."""
    from paged_llm_rs_amd import kernels

    lens = [(0, 700), (7, 3), (block // 2, 260), (0, 1), (block - 1, 2), (3 * block + 1, 95), (0, 33), (0, 31), (0, block), (block // 3, 4)]      # (tokens there already, tokens that come)
    need = [cache.pages_of(a + b, block) for a, b in lens]
    order = torch.randperm(sum(need) + 5).tolist()
    slots, positions = [], []
    for s, (there, comes) in enumerate(lens):
        mine = order[sum(need[:s]):sum(need[:s + 1])]
        slots += [mine[p // block] * block + p % block for p in range(there, there + comes)]
        positions += list(range(there, there + comes))
        if s % 3 == 1:
            slots += [-1] * (5 + s)
            positions += [-1] * (5 + s)
    n = len(slots)
    lib = kernels.library()
    assert lib.pl_qk_norm_rope_kv_write_8bit_tile(n, nkv, block, d) == 32 and lib.pl_qk_norm_rope_kv_write_8bit_waves(n, nkv, block, d) == waves
    qkv = (torch.randn(n, (nq + 2 * nkv) * d, device=cache.DEV) * torch.exp2(3 * torch.randn(n, 1, device=cache.DEV)) * torch.exp2(2 * torch.randn(n, (nq + 2 * nkv) * d, device=cache.DEV))).to(dtype)
    gains = tuple((1 + 0.3 * torch.randn(d, device=cache.DEV)).to(dtype) for _ in range(2)) if normed else (None, None)
    angle = torch.rand(max(positions) + 1, max(rot // 2, 1), device=cache.DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    pages = cache.Pages(len(order), block, nkv, d)
    for pool, power in zip(pages.pools, pages.powers):       # (what earlier steps left: some pages keep their power, some do not)
        pool.copy_((torch.randn(pool.shape, device=cache.DEV) * 60).clamp(-448, 448).to(cache.E4M3))
        power.view(torch.uint8).copy_(torch.randint(112, 130, power.shape, device=cache.DEV))
    before = pages.clone()
    q = torch.full((n, nq * d), -5.0, dtype=dtype, device=cache.DEV)
    at = cache.i32(positions)
    cache.write(pages, qkv, cache.i32(slots), at, nq, q=q, gains=gains, cos=cos, sin=sin, rot=rot, neighbours=neighbours)
    x = qkv.double().view(n, nq + 2 * nkv, d)
    keys = cache.plain_heads(x[:, nq:nq + nkv], gains[1], 1e-6, cos, sin, rot, at, neighbours)
    check_write(pages, before, 0, keys, slots, not normed and not rot)
    check_write(pages, before, 1, x[:, nq + nkv:], slots, True)
    live = at >= 0
    assert bool((q[~live] == -5).all())
    if nq:
        want = cache.plain_heads(x[:, :nq], gains[0], 1e-6, cos, sin, rot, at, neighbours).reshape(n, nq * d)
        allowed = (cache.HALF_BF16 if dtype == torch.bfloat16 else 0) * want.abs() + 1e-5 * want.abs().view(n, nq, d).amax(-1, keepdim=True).expand(n, nq, d).reshape(n, -1)
        assert bool(((q.double() - want).abs() <= allowed)[live].all())
    # in place
    twin, again = before.clone(), qkv.clone()
    cache.write(twin, again, cache.i32(slots), at, nq, gains=gains, cos=cos, sin=sin, rot=rot, neighbours=neighbours)
    assert torch.equal(again[live, :nq * d], q[live]) and torch.equal(again[:, nq * d:], qkv[:, nq * d:]) and torch.equal(again[~live], qkv[~live])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(twin, pages))


def test_the_most_requests_of_a_step():
    """8,192 requests, which take all the room that the kernel has for their sums, with pages from a list of free ones and without."""
    requests = 8192
    ctx = [1 + (7 * s) % 50 for s in range(requests)]
    q_len = [c if s % 5 == 0 else 1 for s, c in enumerate(ctx)]
    ctx[17], q_len[17] = 0, 3
    table = [[4 * s + i for i in range(4)] for s in range(requests)]
    free = list(range(4 * requests, 4 * requests + 9000))
    cache.check_tables(q_len, ctx, table, 16, free, sum(q_len) + 11)
    cache.check_tables(q_len, ctx, table, 16, None, sum(q_len) + 11)
