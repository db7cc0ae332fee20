"""The operators of a paged cache held in 8 bits, each against a plain implementation in 64 bits (or whole numbers), and a run of them together."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
HALF_BF16, HALF_F32, HALF_E4M3 = 2.0 ** -8, 2.0 ** -24, 2.0 ** -4


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pages_of(tokens, block):
    return -(-tokens // block)


# ---- block tables and slots -----------------------------------------------------------------------------------------------

def plain_tables(q_len, ctx, table, block, free, rows):
    """Whole numbers, request by request."""
    table = [list(r) for r in table]
    width = len(table[0])
    positions, seq_of, slots, q_start, taken, at = [], [], [], [], 0, 0
    for s, (q, c) in enumerate(zip(q_len, ctx)):
        q_start.append(at)
        at += q
        idle = c < q or c <= 0
        held = 0 if idle else min(pages_of(c - q, block), width)
        need = 0 if idle else min(pages_of(c, block), width)
        if free is not None:
            for i in range(held, width):
                table[s][i] = -1
                if i < need:
                    table[s][i] = free[taken] if taken < len(free) else -1
                    taken += 1
        for i in range(q):
            p = c - q + i if c >= q else -1
            page = table[s][p // block] if p >= 0 and p // block < width else -1
            positions.append(p)
            seq_of.append(s)
            slots.append(page * block + p % block if page >= 0 else -1)
    positions += [-1] * (rows - at)
    slots += [-1] * (rows - at)
    seq_of += [len(q_len) - 1] * (rows - at)
    return table, positions[:rows], seq_of[:rows], slots[:rows], q_start, [taken]


def check_tables(q_len, ctx, table, block, free, rows):
    from paged_llm_rs_amd import kernels

    want = plain_tables(q_len, ctx, table, block, free, rows)
    t = i32(table)
    made = kernels.step_tables(i32(q_len), i32(ctx), t, block, None if free is None else i32(free), rows)
    got = (t.tolist(), made.positions.tolist(), made.seq_of.tolist(), made.slots.tolist(), made.q_start.tolist(), made.pages.tolist())
    for a, b, what in zip(got, want, ("table", "positions", "seq_of", "slots", "q_start", "pages")):
        assert a == b, what


@pytest.mark.parametrize("block", [1, 5, 16, 128])
@pytest.mark.parametrize("seqs", [1, 3, 63, 64, 65, 255, 257, 700])
def test_step_tables(block, seqs):
    g = torch.Generator().manual_seed(seqs * 1000 + block)

    def draw(low, high):
        return int(torch.randint(low, high + 1, (1,), generator=g))

    ctx = [draw(0, 60) for _ in range(seqs)]
    q_len = [draw(0, c) if draw(0, 3) else min(c, 1) for c in ctx]
    if seqs > 2:
        ctx[1], q_len[1] = 0, 4                         # rows that a step is padded with, in the middle of it
    width = max(1, pages_of(60, block) + 1)
    pages = seqs * width
    order = torch.randperm(2 * pages, generator=g).tolist()
    table = [order[s * width:(s + 1) * width] for s in range(seqs)]     # (entries behind the held ones are anybody's)
    free = order[pages:]
    for rows in (sum(q_len), sum(q_len) + 37):
        check_tables(q_len, ctx, table, block, free, rows)
        check_tables(q_len, ctx, table, block, None, rows)


def test_step_tables_that_lack_pages_or_room():
    # too few free pages, none at all, a table that is too narrow, a page that was given back
    check_tables([5, 20, 7], [5, 20, 40], [[-1, -1, -1]] * 3, 16, [9, 8], 32)
    check_tables([5, 20, 7], [5, 20, 40], [[-1, -1, -1]] * 3, 16, [], 32)
    check_tables([5, 60], [5, 60], [[-1, -1]] * 2, 16, [9, 8, 7, 6, 5], 70)
    check_tables([1, 1], [33, 34], [[-1, -1, 3, 4]] * 2, 16, None, 2)
    check_tables([0], [0], [[-1]], 16, [1], 0)
    check_tables([1] * 4, [2 ** 20, 2 ** 20 + 1, 1, 17], [[7] * (2 ** 16 + 1)] * 4, 16, [1, 2, 3], 4)


# ---- the write --------------------------------------------------------------------------------------------------------------

def least_power(top):
    """The byte of the least power of two whose 448-fold holds top (64-bit, not negative)."""
    if top == 0:
        return 1
    part, exponent = math.frexp(top)
    return max(exponent - 9 + (1 if part > 0.875 else 0), -126) + 127


def plain_heads(x, gain, eps, cos, sin, rot, positions, neighbours):
    """Norm and rotation in 64 bits; x [rows, heads, d]."""
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    if rot:
        c, s = (t.double()[positions.long().clamp(0, t.shape[0] - 1)].unsqueeze(1) for t in (cos, sin))
        x = x.clone()
        a, b = (x[..., 0:rot:2].clone(), x[..., 1:rot:2].clone()) if neighbours else (x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone())
        first, second = a * c - b * s, b * c + a * s
        if neighbours:
            x[..., 0:rot:2], x[..., 1:rot:2] = first, second
        else:
            x[..., :rot // 2], x[..., rot // 2:rot] = first, second
    return x


class Pages:
    def __init__(self, pages, block, nkv, d, fill=0x7f, power=0xff):
        self.block, self.nkv, self.d = block, nkv, d
        self.pools = [torch.full((pages * block, nkv * d), fill, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
        self.powers = [torch.full((pages, nkv), power, dtype=torch.uint8, device=DEV).view(E8M0) for _ in range(2)]

    def __iter__(self):
        return iter((*self.pools, *self.powers))

    def clone(self):
        c = object.__new__(Pages)
        c.__dict__.update(self.__dict__)
        c.pools, c.powers = [p.clone() for p in self.pools], [p.clone() for p in self.powers]
        return c


def write(pages, qkv, slots, positions, nq, q=None, gains=(None, None), eps=1e-6, cos=None, sin=None, rot=0, **more):
    from paged_llm_rs_amd import kernels

    k, v, ks, vs = pages
    kernels.qk_norm_rope_kv_write_8bit(qkv, q, *gains, eps, cos, sin, rot, positions, slots, pages.block, k, v, ks, vs, nq, pages.nkv, pages.d, **more)


def check_rows(pages, which, want, slots, live_rows, before, f32):
    """The rows in their slots, as values, against ``want`` [rows, nkv, d] in 64 bits: a rounding to e4m3 is half a step, 2^-4 of the value, or 2^-10 units below the smallest normal
    one; the 32-bit arithmetic before it is off by less than 1e-5 of the row's largest.  Everything else in the pool is as it was."""
    nkv, d, block = pages.nkv, pages.d, pages.block
    held = pages.pools[which].double().cpu().view(-1, nkv, d)
    unit = torch.exp2(pages.powers[which].view(torch.uint8).double().cpu() - 127)
    want = want.cpu()
    for r in live_rows:
        u = unit[slots[r] // block].view(nkv, 1)
        off = (held[slots[r]] * u - want[r]).abs()
        allowed = torch.maximum(HALF_E4M3 * want[r].abs(), 2.0 ** -10 * u) + 1e-5 * want[r].abs().amax(-1, keepdim=True)
        assert bool((off <= allowed).all()), (which, r, float((off / allowed).max()))
    touched = torch.zeros(held.shape[0], dtype=torch.bool)
    touched[[slots[r] for r in live_rows]] = True
    now, then = (p.pools[which].view(torch.uint8).cpu() for p in (pages, before))
    assert torch.equal(now[~touched], then[~touched])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d,block,rot,normed,neighbours", [
    (16, 8, 128, 16, 128, True, False), (12, 4, 64, 16, 32, False, False), (6, 2, 80, 32, 80, True, False), (8, 4, 256, 128, 128, True, False), (4, 4, 32, 5, 30, True, False),
    (5, 5, 16, 1, 16, True, True), (8, 1, 96, 64, 0, True, False), (3, 1, 176, 16, 22, False, True), (0, 3, 48, 16, 0, False, False)])
def test_fresh_rows_into_their_pages(dtype, nq, nkv, d, block, rot, normed, neighbours):
    lens = [1, 2 * block + 3, block, 5 * block + 1, 3]
    n = sum(lens) + 2
    need = [pages_of(c, block) for c in lens]
    order = torch.randperm(sum(need) + 3).tolist()
    slots, positions = [], []
    for s, c in enumerate(lens):
        mine = order[sum(need[:s]):sum(need[:s + 1])]
        slots += [mine[p // block] * block + p % block for p in range(c)]
        positions += list(range(c))
    slots += [-1, -1]
    positions += [-1, -1]
    # rows of unlike size, values between them whose sizes span more than e4m3 holds, a row of zeros
    qkv = (torch.randn(n, (nq + 2 * nkv) * d, device=DEV) * torch.exp2(4 * torch.randn(n, 1, device=DEV)) * torch.exp2(3 * torch.randn(n, (nq + 2 * nkv) * d, device=DEV))).to(dtype)
    qkv[2] = 0
    gains = tuple((1 + 0.3 * torch.randn(d, device=DEV)).to(dtype) for _ in range(2)) if normed else (None, None)
    angle = torch.rand(max(lens), max(rot // 2, 1), device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    pages = Pages(len(order), block, nkv, d)
    before, original = pages.clone(), qkv.clone()
    q = torch.full((n, nq * d), -5.0, dtype=dtype, device=DEV)
    at = i32(positions)
    write(pages, qkv, i32(slots), at, nq, q=q, gains=gains, cos=cos, sin=sin, rot=rot, neighbours=neighbours)
    x = original.double().view(n, nq + 2 * nkv, d)
    assert torch.equal(qkv, original)
    live = list(range(n - 2))
    for which, (rows, gain, turn) in enumerate(((x[:, nq:nq + nkv], gains[1], rot), (x[:, nq + nkv:], None, 0))):
        want = plain_heads(rows, gain, 1e-6, cos, sin, turn, at, neighbours)
        check_rows(pages, which, want, slots, live, before, dtype == torch.float32)
        # the powers: least ones, of the values as 32 bits have them (a maximum within 1e-5 of a border may fall on either side)
        got = pages.powers[which].view(torch.uint8).cpu()
        for page in {s // block for s in slots if s >= 0}:
            top = want[[r for r in live if slots[r] // block == page]].abs().amax((0, 2)).tolist()
            for h in range(nkv):
                assert least_power(top[h] * (1 - 1e-5)) <= int(got[page, h]) <= least_power(top[h] * (1 + 1e-5))
        unused = [p for p in range(len(order)) if p not in {s // block for s in slots if s >= 0}]
        assert bool((got[unused] == 0xff).all())
    want = plain_heads(x[:, :nq], gains[0], 1e-6, cos, sin, rot, at, neighbours).reshape(n, nq * d)
    assert bool((q[-2:] == -5).all())
    if nq:
        # one rounding to the type, and 32-bit sums and products of which a value has a dozen, none larger than the row's largest value
        allowed = (HALF_BF16 if dtype == torch.bfloat16 else 0) * want.abs() + 1e-5 * want.abs().view(n, nq, d).amax(-1, keepdim=True).expand(n, nq, d).reshape(n, -1)
        assert bool(((q.double() - want).abs() <= allowed)[:-2].all())
    # in place, and the queries alone
    again = original.clone()
    twin = before.clone()
    write(twin, again, i32(slots), at, nq, gains=gains, cos=cos, sin=sin, rot=rot, neighbours=neighbours)
    assert torch.equal(again[:-2, :nq * d], q[:-2]) and torch.equal(again[:, nq * d:], original[:, nq * d:]) and torch.equal(again[-2:], original[-2:])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(twin, pages))
    again = original.clone()
    twin = before.clone()
    write(twin, again, i32(slots), at, nq, gains=gains, cos=cos, sin=sin, rot=rot, neighbours=neighbours, write_kv=False)
    assert torch.equal(again[:-2, :nq * d], q[:-2]) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(twin, before))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block,steps", [(16, [1] * 20), (16, [3, 1, 2, 11, 30, 1]), (5, [2, 2, 2, 7]), (128, [1, 100, 40, 1, 1]), (300, [290, 7, 20])])
def test_a_page_that_grows_while_it_fills(dtype, block, steps):
    """Values take no arithmetic on the way, so the bytes are those of a plain simulation: the power grows, what is there is rounded again."""
    nkv, d = 3, 48
    pages = Pages(8, block, nkv, d)
    mine, total = [5, 2, 7, 0, 1], 0
    want, powers = {}, {}
    for i, count in enumerate(steps):
        rows = (torch.randn(count, 2 * nkv * d, device=DEV) * torch.exp2(torch.randn(count, 1, device=DEV) * 3 + i / 4)).to(dtype)
        slots = [mine[p // block] * block + p % block for p in range(total, total + count)]
        write(pages, rows, i32(slots), i32(list(range(total, total + count))), 0)
        v = rows.float().cpu().view(count, 2, nkv, d)[:, 1]
        for page in sorted({s // block for s in slots}, key=mine.index):
            inside = [r for r in range(count) if slots[r] // block == page]
            for h in range(nkv):
                fresh = slots[inside[0]] % block == 0
                had = 0 if fresh else powers[page, h]
                power = max(least_power(float(v[inside, h].abs().max())), had)
                if not fresh and power > had:
                    for o in range(slots[inside[0]] % block):
                        want[page * block + o, h] = torch.ldexp(want[page * block + o, h].float(), torch.tensor(had - power)).to(E4M3)
                for r in inside:
                    want[slots[r], h] = torch.ldexp(v[r, h], torch.tensor(127 - power)).to(E4M3)
                powers[page, h] = power
        total += count
    got, unit = pages.pools[1].cpu().view(-1, nkv, d), pages.powers[1].view(torch.uint8).cpu()
    for (slot, h), x in want.items():
        assert torch.equal(got[slot, h].view(torch.uint8), x.view(torch.uint8)), (slot, h)
    for (page, h), power in powers.items():
        assert int(unit[page, h]) == power


def test_values_that_are_not_finite_and_the_ends_of_the_range():
    nkv, d, block = 1, 16, 16
    top = torch.finfo(torch.float32).max
    rows = torch.zeros(6, 2 * d, device=DEV)
    rows[0, d:d + 4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    rows[1, d:d + 2] = torch.tensor([448.0, -1.0])
    rows[2, d:d + 2] = torch.tensor([448.5, 1.0])                          # past 448: the next power
    rows[3, d:d + 2] = torch.tensor([top, -top])
    rows[4, d:d + 2] = torch.tensor([2.0 ** -130, -2.0 ** -149])           # below the smallest power's smallest value
    pages = Pages(6, block, nkv, d)
    write(pages, rows, i32([block * i for i in range(6)]), i32([0] * 6), 0)
    power = pages.powers[1].view(torch.uint8).cpu().view(-1).tolist()
    value = (pages.pools[1].double().cpu()[::block] * torch.exp2(torch.tensor(power, dtype=torch.float64) - 127).view(-1, 1))
    assert power == [least_power(3.0), 127, 128, least_power(top), 1, 1]
    assert value[0, :3].isnan().all() and value[0, 3] == 3
    assert value[1, :2].tolist() == [448, -1] and value[2, :2].tolist() == [448, 1]
    assert value[3, 0] == 2.0 ** 128 and value[3, 1] == -(2.0 ** 128)      # (rounded up to a power of two: 256 times its unit)
    assert value[4, :2].tolist() == [2.0 ** -130, 0.0] and value[5].abs().max() == 0


# ---- attention -----------------------------------------------------------------------------------------------------------------

class Scene:
    """Requests over shuffled pages.  Everything that no row sees is NaN: other pages and their powers, slots behind a context."""

    def __init__(self, requests, nq, nkv, d, block, dtype, extra_rows=0, largest=4.0):
        self.requests, self.nq, self.nkv, self.d, self.block = requests, nq, nkv, d, block
        need = [pages_of(max(c, 0), block) for _, c in requests]
        total = sum(need) + 3
        order = torch.randperm(total).tolist()
        self.width = max(max(need), 1) + 2
        table = torch.full((len(requests), self.width), -1, dtype=torch.int32)
        self.pages = Pages(total, block, nkv, d)
        pools = [p.view(torch.uint8) for p in self.pages.pools]
        self.values = []
        for s, (q, c) in enumerate(requests):
            mine = order[sum(need[:s]):sum(need[:s + 1])]
            table[s, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            kv = []
            for which in range(2):
                bytes_ = (torch.randn(max(c, 0), nkv * d, device=DEV) * 60).clamp(-448, 448).to(E4M3)
                powers = torch.randint(127 - 8, 127 - 5, (len(mine), nkv), device=DEV).to(torch.uint8)
                if mine:
                    self.pages.powers[which].view(torch.uint8)[mine] = powers
                    slots = torch.tensor([mine[p // block] * block + p % block for p in range(c)], device=DEV)
                    pools[which][slots] = bytes_.view(torch.uint8)
                    unit = torch.exp2(powers.double() - 127).repeat_interleave(block, 0)[:c]
                    kv.append(bytes_.double().view(c, nkv, d) * unit.unsqueeze(-1))
                else:
                    kv.append(torch.zeros(0, nkv, d, dtype=torch.float64, device=DEV))
            self.values.append(kv)
        self.table = table.to(DEV)
        brings = [q for q, _ in requests]
        self.q_len, self.ctx_len = i32(brings), i32([c for _, c in requests])
        self.starts = [sum(brings[:s]) for s in range(len(brings))]
        self.q_start = i32(self.starts)
        self.n = sum(brings) + extra_rows
        self.stride = nq * d + 16
        self.q = (torch.randn(self.n, self.stride, device=DEV) * largest / 4).to(dtype)
        self.scale = d ** -0.5

    def run(self, window=0, out=None, **more):
        from paged_llm_rs_amd import kernels

        if out is None:
            out = torch.full((self.n, self.nq * self.d), -7.0, dtype=self.q.dtype, device=DEV)
        k, v, ks, vs = self.pages
        live = [q for q, c in self.requests if c >= q]
        more.setdefault("min_q_len", min(live))
        kernels.paged_attention_8bit(self.q, self.stride, out, self.q_start, self.q_len, self.ctx_len, max([q for q, _ in self.requests]), more.pop("max_ctx", max(c for _, c in self.requests)),
                                     self.table, self.block, k, v, ks, vs, self.nq, self.nkv, self.d, self.scale, window, **more)
        return out

    def check(self, out, window=0):
        """Per value, with A = sum p |v| / sum p: bfloat16 rounds every weight (2^-8 A) and the result (2^-8 of it).  32-bit sums: a score is off by (d + 16) halves of a last place of
        sum |q k| scale (three times as many additions in 32 bits), which moves its weight by as much, and so the result by twice that times A; the sums over keys pass one addition for
        eight keys (and one for every share and wave), each off by half a last place of what they hold."""
        group, bf16 = self.nq // self.nkv, self.q.dtype == torch.bfloat16
        untouched = torch.ones(self.n, dtype=torch.bool, device=DEV)
        for (q, c), at, (k, v) in zip(self.requests, self.starts, self.values):
            if q == 0 or c < q:
                continue
            untouched[at:at + q] = False
            pos = torch.arange(c - q, c, device=DEV).view(-1, 1)
            key = torch.arange(c, device=DEV).view(1, -1)
            seen = key <= pos
            if window > 0:
                seen &= key > pos - window
            if window < 0:
                seen &= key >= pos - pos % -window
            x = self.q[at:at + q, :self.nq * self.d].double().view(q, self.nkv, group, self.d)
            for h in range(self.nkv):
                score = (x[:, h].reshape(q * group, self.d) @ k[:, h].T * self.scale).view(q, group, c)
                size = (x[:, h].abs().reshape(q * group, self.d) @ k[:, h].abs().T * self.scale).view(q, group, c)
                mask = ~seen.view(q, 1, c)
                p = torch.softmax(score.masked_fill(mask, -math.inf), -1)
                want, A = p @ v[:, h], p @ v[:, h].abs()
                off = size.masked_fill(mask, 0).amax(-1, keepdim=True) * (self.d + 16) * (1 if bf16 else 3) * HALF_F32
                allowed = A * (2 * off + (c / 8 + 64) * HALF_F32)
                allowed = allowed + (HALF_BF16 * (A + want.abs()) if bf16 else HALF_F32 * want.abs())
                got = out[at:at + q].double().view(q, self.nkv, group, self.d)[:, h]
                assert bool(((got - want).abs() <= allowed).all()), (q, c, h, float(((got - want).abs() / allowed).nan_to_num(1e9).max()))
        assert bool((out[untouched] == -7).all())


HEADS = [(16, 8, 128), (8, 1, 128), (4, 4, 32), (6, 2, 80), (8, 4, 256), (12, 12, 96), (5, 5, 16), (40, 1, 64), (7, 1, 176), (64, 8, 128)]
MIXES = {
    "one": [(1, 1)],
    "singles": [(1, 1), (1, 2), (1, 17), (1, 700), (1, 33), (1, 16), (1, 513)],
    "drafts": [(5, 5), (2, 130), (9, 1100), (5, 512)],
    "prompts": [(130, 130), (1, 1), (70, 70), (33, 33)],
    "portions": [(65, 600), (1, 90), (200, 1333), (0, 40), (1, 1), (3, 3)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mix", sorted(MIXES))
@pytest.mark.parametrize("nq,nkv,d", HEADS)
def test_attention(dtype, mix, nq, nkv, d):
    scene = Scene(MIXES[mix], nq, nkv, d, 16, dtype, extra_rows=3)
    scene.check(scene.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 7, 300, -1, -64, -100])
@pytest.mark.parametrize("mix", ["singles", "drafts", "portions"])
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (6, 2, 80)])
def test_attention_under_a_window(dtype, window, mix, nq, nkv, d):
    scene = Scene(MIXES[mix], nq, nkv, d, 16, dtype)
    scene.check(scene.run(window), window)


@pytest.mark.parametrize("block", [1, 5, 32, 128, 1000])
@pytest.mark.parametrize("mix", ["singles", "portions"])
def test_attention_over_pages_of_other_sizes(block, mix):
    for dtype in (torch.bfloat16, torch.float32):
        scene = Scene(MIXES[mix], 8, 2, 64, block, dtype)
        scene.check(scene.run())
        scene.check(scene.run(40), 40)


def test_attention_leaves_padding_rows_and_says_a_context_that_is_too_long():
    scene = Scene([(3, 40), (9, 0), (1, 600), (4, 3)], 4, 2, 64, 16, torch.bfloat16, extra_rows=2)
    out = scene.run(min_q_len=0)
    scene.check(out)
    long = scene.run(max_ctx=40, min_q_len=0)
    assert bool(long[12].isnan().all()) and torch.equal(long[:3], out[:3])
    far = scene.run(max_ctx=100000, min_q_len=0)       # (a bound that is far from every context)
    scene.check(far)


UNLIKE = [(1, 1), (1, 5000), (2, 2), (1, 1100), (3, 2300), (0, 40), (1, 4097), (4, 3), (2, 1024), (1, 1025), (3, 700), (1, 3333)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(64, 64, 16), (384, 64, 32), (6, 2, 80)])
def test_attention_of_more_shares_than_the_chip_holds(dtype, nq, nkv, d):
    """Contexts so unlike, or said to be so long, that the kernel of few rows cuts them itself."""
    scene = Scene(UNLIKE, nq, nkv, d, 16, dtype, extra_rows=2)
    scene.check(scene.run(min_q_len=0))
    scene.check(scene.run(min_q_len=0, max_ctx=300000))
    for window in (2500, -3000):
        scene.check(scene.run(window, min_q_len=0, max_ctx=300000), window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests", [[(1 + s % 5, 1100 + 37 * s) for s in range(60)], [(1, 2500 + s) for s in range(64)], [(1, 900 + 31 * s) for s in range(65)]])
def test_attention_of_full_rounds_of_shares(dtype, requests):
    scene = Scene(requests, 64 if requests[1][0] == 2 else 16, 8, 64, 16, dtype)
    scene.check(scene.run())


def test_contexts_that_are_too_long_among_shares_that_the_kernel_cuts():
    scene = Scene(UNLIKE, 64, 64, 16, 16, torch.bfloat16)
    out, long = scene.run(min_q_len=0), scene.run(min_q_len=0, max_ctx=2048)
    for (q, c), at in zip(scene.requests, scene.starts):
        if c > 2048:
            assert bool(long[at:at + q].isnan().all())
            long[at:at + q] = out[at:at + q]
    scene.check(long)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_large_and_of_equal_scores(dtype):
    scene = Scene([(1, 900), (40, 300)], 8, 2, 64, 16, dtype, largest=200.0)        # weights of one and of zero
    scene.check(scene.run())
    scene = Scene([(1, 900), (40, 300)], 8, 2, 64, 16, dtype)
    scene.q.zero_()
    scene.check(scene.run())


def test_attention_on_another_stream_and_in_graphs():
    """Two captured graphs and eager calls in turn, on one state: every replay gives the eager result."""
    scene = Scene(MIXES["portions"], 16, 8, 128, 16, torch.bfloat16)
    want = scene.run()
    scene.check(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(scene.run(), want)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for window in (0, 50):
        out = torch.full_like(want, -7.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scene.run(window, out=out)
        graphs.append(graph)
        outs.append(out)
    narrow = scene.run(50)
    for _ in range(4):
        for out in outs:
            out.fill_(-7.0)
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(scene.run(), want)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], narrow)


# ---- together -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_requests_from_their_first_token_on(dtype):
    """Prompts, portions, drafts and single tokens, pages from a list of free ones, written and read: every step's rows against attention over the keys and values that the
    cache holds, and what it holds against what was written."""
    from paged_llm_rs_amd import kernels

    nq, nkv, d, block, eps = 8, 2, 64, 16, 1e-6
    S, width, total = 4, 12, 48
    table = torch.full((S, width), -1, dtype=torch.int32, device=DEV)
    free = i32(torch.randperm(total).tolist())
    pages = Pages(total, block, nkv, d)
    gains = tuple((1 + 0.1 * torch.randn(d, device=DEV)).to(dtype) for _ in range(2))
    angle = torch.rand(block * width, d // 2, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    ctx, handed = [0] * S, 0
    kept = [[torch.zeros(0, nkv, d, dtype=torch.float64, device=DEV) for _ in range(2)] for _ in range(S)]
    for brings in ([20, 0, 7, 33], [1, 40, 1, 1], [1, 1, 5, 1], [16, 1, 1, 1], [1, 1, 1, 30], [1, 1, 1, 1]):
        ctx = [c + b for c, b in zip(ctx, brings)]
        n = sum(brings)
        made = kernels.step_tables(i32(brings), i32(ctx), table, block, free[handed:], n)
        handed += int(made.pages)
        assert handed == sum(pages_of(c, block) for c in ctx)
        qkv = (torch.randn(n, (nq + 2 * nkv) * d, device=DEV) * torch.exp2(torch.randn(n, 1, device=DEV))).to(dtype)
        q = torch.empty(n, nq * d, dtype=dtype, device=DEV)
        write(pages, qkv, made.slots, made.positions, nq, q=q, gains=gains, cos=cos, sin=sin, rot=d)
        out = torch.full_like(q, -7.0)
        kernels.paged_attention_8bit(q, nq * d, out, made.q_start, i32(brings), i32(ctx), max(brings), max(ctx), table, block, *pages, nq, nkv, d, d ** -0.5, min_q_len=min(brings))
        scene = object.__new__(Scene)
        scene.requests, scene.nq, scene.nkv, scene.d, scene.q, scene.n, scene.scale = list(zip(brings, ctx)), nq, nkv, d, q, n, d ** -0.5
        scene.starts = made.q_start.tolist()
        scene.values = []
        x = qkv.double().view(n, nq + 2 * nkv, d)
        wrote = (plain_heads(x[:, nq:nq + nkv], gains[1], eps, cos, sin, d, made.positions, False), x[:, nq + nkv:])
        for s in range(S):
            at = scene.starts[s]
            held = []
            for which in range(2):
                kept[s][which] = torch.cat([kept[s][which], wrote[which][at:at + brings[s]]])
                place = torch.arange(ctx[s], device=DEV)
                page = table[s, place // block].long()
                unit = torch.exp2(pages.powers[which].view(torch.uint8).double()[page] - 127).unsqueeze(-1)
                held.append(pages.pools[which].double().view(-1, nkv, d)[page * block + place % block] * unit)
                # (rounded at most once in every unit it has had: half a step of each, together less than a step of the last)
                off = (held[-1] - kept[s][which]).abs()
                assert bool((off <= torch.maximum(2 * HALF_E4M3 * kept[s][which].abs(), 2.0 ** -9 * unit) + 1e-5).all())
            scene.values.append(held)
        scene.check(out)


def test_a_captured_step_of_all_three():
    """Slots, write and attention of a decoding step in one graph, replayed while the contexts grow, with eager work between: the bits of the eager calls on pages of their own."""
    from paged_llm_rs_amd import kernels

    nq, nkv, d, block, S, width = 16, 8, 128, 16, 5, 40
    ctx = i32([600, 17, 16, 1, 333])
    brings = i32([1] * S)
    table = i32(torch.randperm(S * width).tolist()).view(S, width)
    pages = Pages(S * width, block, nkv, d, fill=0x30, power=121)
    qkv = torch.randn(S, (nq + 2 * nkv) * d, device=DEV).to(torch.bfloat16)
    gain = torch.ones(d, dtype=torch.bfloat16, device=DEV)
    angle = torch.rand(block * width, d // 2, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()

    def step(pages, ctx, qkv, q, out):
        made = kernels.step_tables(brings, ctx, table, block, None, S)
        write(pages, qkv, made.slots, made.positions, nq, q=q, gains=(gain, gain), cos=cos, sin=sin, rot=d)
        kernels.paged_attention_8bit(q, nq * d, out, made.q_start, brings, ctx, 1, block * width, table, block, *pages, nq, nkv, d, d ** -0.5)

    twin = pages.clone()
    q, out = (torch.empty(S, nq * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    idle = torch.zeros_like(ctx)
    step(pages, idle, qkv, q, out)                        # (a step of padding: nothing is written)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pages, twin))
    static = ctx.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pages, static, qkv, q, out)
    for i in range(20):
        qkv.copy_((torch.randn(S, (nq + 2 * nkv) * d, device=DEV) * 2 ** (i / 4)).to(torch.bfloat16))
        static.copy_(ctx + i)
        graph.replay()
        q2, out2 = torch.empty_like(q), torch.empty_like(out)
        step(twin, ctx + i, qkv, q2, out2)
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(out, out2), i
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pages, twin)), i


def test_pages_behind_four_gigabytes():
    """The same requests over the last pages of pools of 4.9 GB: the bits of a small pool."""
    from paged_llm_rs_amd import kernels

    scene = Scene(MIXES["portions"], 16, 8, 128, 16, torch.bfloat16)
    want = scene.run()
    total, few = 300000, scene.pages.powers[0].shape[0]
    far = Pages(total, 16, 8, 128)
    for big, small in zip(far, scene.pages):
        big.view(torch.uint8)[-small.shape[0]:] = small.view(torch.uint8)
    table = torch.where(scene.table >= 0, scene.table + (total - few), scene.table)
    near = scene.pages
    scene.pages, scene.table = far, table
    assert torch.equal(scene.run(), want)
    qkv = torch.randn(40, (4 + 2 * 8) * 128, device=DEV).to(torch.bfloat16)
    slots = i32([3 * 16 + 5 + i for i in range(40)])
    write(near, qkv, slots, i32(list(range(40))), 4)
    write(far, qkv, slots + (total - few) * 16, i32(list(range(40))), 4)
    for big, small in zip(far, near):
        assert torch.equal(big.view(torch.uint8)[-small.shape[0]:], small.view(torch.uint8))
    made = kernels.step_tables(scene.q_len, scene.ctx_len, table, 16, None, scene.n)
    assert int(made.slots.max()) >= (total - few) * 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_many_heads_a_key_head_and_of_a_long_context(dtype):
    scene = Scene([(1, 300), (2, 70), (1, 1)], 300, 1, 16, 16, dtype)
    scene.check(scene.run())
    scene = Scene([(1, 33000), (3, 20000), (1, 12)], 8, 1, 64, 64, dtype)
    scene.check(scene.run())


# ---- refusals --------------------------------------------------------------------------------------------------------------------

def test_refusals():
    from paged_llm_rs_amd import kernels
    from paged_llm_rs_amd.errors import TensorError

    scene = Scene([(2, 20), (1, 5)], 4, 2, 64, 16, torch.bfloat16)
    k, v, ks, vs = scene.pages
    out = torch.empty(scene.n, 4 * 64, dtype=torch.bfloat16, device=DEV)

    def attend(**other):
        a = dict(q=scene.q, q_row_stride=scene.stride, out=out, q_start=scene.q_start, q_len=scene.q_len, ctx_len=scene.ctx_len, max_q_len=2, max_ctx=20, block_table=scene.table,
                 block_size=16, k_pool=k, v_pool=v, k_scale=ks, v_scale=vs, nq=4, nkv=2, d=64, scale=0.1)
        a.update(other)
        kernels.paged_attention_8bit(**a)

    attend()
    for other in (dict(q=scene.q.half()), dict(q=scene.q[:, 8:]), dict(q_row_stride=200), dict(out=out.float()), dict(out=out[:2]), dict(q_start=scene.q_start[:1]),
                  dict(q_len=scene.q_len.long()), dict(ctx_len=scene.ctx_len.cpu()), dict(max_q_len=0), dict(max_q_len=4), dict(min_q_len=3), dict(max_ctx=0), dict(block_table=scene.table[0]),
                  dict(block_size=7), dict(block_size=0), dict(k_pool=k.view(torch.uint8)), dict(v_pool=v[:16]), dict(k_scale=ks.view(torch.uint8)), dict(v_scale=vs[:1]), dict(nq=3), dict(nkv=3),
                  dict(d=72), dict(d=8), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises(TensorError):
            attend(**other)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(30, 32, device=DEV)
    gain = torch.ones(64, dtype=torch.bfloat16, device=DEV)

    def put(**other):
        a = dict(qkv=qkv, q=out, q_gain=gain, k_gain=gain, eps=1e-6, cos=table, sin=table, rot=64, positions=i32([0, 1, 2]), slots=i32([0, 1, 2]), block_size=16, k_pool=k, v_pool=v,
                 k_scale=ks, v_scale=vs, nq=4, nkv=2, d=64)
        a.update(other)
        kernels.qk_norm_rope_kv_write_8bit(**a)

    put()
    for other in (dict(qkv=qkv.half()), dict(qkv=qkv[:, :-64]), dict(q=out.float()), dict(q_gain=None), dict(k_gain=gain.float()), dict(q_gain=gain[:8]), dict(cos=table[:, :8]), dict(sin=table[:3]),
                  dict(cos=table.double()), dict(rot=63), dict(rot=66), dict(rot=-2), dict(positions=i32([0, 1])), dict(slots=i32([0, 1, 2]).long()), dict(block_size=15), dict(k_pool=v.float()),
                  dict(v_scale=ks.view(torch.uint8)), dict(d=32)):
        with pytest.raises(TensorError):
            put(**other)

    def lay(**other):
        a = dict(q_len=scene.q_len, ctx_len=scene.ctx_len, block_table=scene.table, block_size=16, free_pages=None, rows=3)
        a.update(other)
        kernels.step_tables(**a)

    lay()
    for other in (dict(q_len=scene.q_len.long()), dict(q_len=scene.q_len[:0]), dict(ctx_len=scene.ctx_len[:1]), dict(block_table=scene.table[:1]), dict(block_table=scene.table[:, :0]), dict(block_size=0),
                  dict(rows=-1), dict(free_pages=scene.q_len.long()), dict(free_pages=scene.q_len.cpu()), dict(q_len=scene.q_len.cpu())):
        with pytest.raises(TensorError):
            lay(**other)
    many = torch.ones(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(TensorError):
        kernels.step_tables(many, many, many.view(-1, 1), 16, None, 8193)
