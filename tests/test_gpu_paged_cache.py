"""The paged cache in 4 bits -- append, read, attention -- against the 64-bit oracle."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged_cache as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def tables(rows, dim):
    angle = torch.outer(torch.arange(rows, dtype=torch.float64), 100.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2)))
    angle = torch.cat([angle, angle], 1)
    return angle.sin().float(), angle.cos().float()


def layout(batch, tokens, page, seed, spare=2):
    """(page table in no order, pages)."""
    per = max(1, -(-tokens // page))
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(batch * per + spare, generator=g)[:batch * per].view(batch, per).int(), batch * per + spare


class Both:
    """A cache on the GPU and the oracle's pages, written together."""

    def __init__(self, vgo, device, pages, kv_heads, page, dim, masses=False):
        self.vgo, self.device, self.masses = vgo, device, masses
        self.cache = vgo.PagedCache.empty(pages, kv_heads, dim, page_size=page, masses=masses, device=device)
        self.pages = oracle.Pages(pages, kv_heads, page, dim)

    def to(self, t):
        return t.to(self.device) if isinstance(t, torch.Tensor) else None if t is None else tuple(x.to(self.device) for x in t)

    def append(self, k, v, table, starts, counts=None, q=None, rope=None, positions=None, log_mass=None):
        got = self.vgo.cache_append(self.cache, self.to(k), self.to(v), self.to(table), self.to(starts), self.to(counts),
                                    q=self.to(q), rope=self.to(rope), positions=self.to(positions), log_mass=self.to(log_mass))
        want = oracle.append(self.pages, k, v, table, starts, counts, q=q, rope=rope, positions=positions, log_mass=log_mass)
        if q is not None:
            got = got.double().cpu()
            # One product and one sum in fp32 (2^-24 of each; together less than 2^-23 of the parts' magnitudes, which
            # rotation by an orthogonal pair bounds by its two channels'), then half a step of the type; the smallest normal
            # number of the type for what rounds to less.
            parts = q.double().abs() + q.double().abs().roll(q.shape[-1] // 2, -1)
            off = torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -23 * parts + torch.finfo(q.dtype).tiny
            assert ((got - want).abs() <= off).all()
        return got

    def check_everything(self):
        """Every place of every page, and the masses."""
        pages, page = self.cache.data.shape[0], self.cache.page_size
        table = torch.arange(pages, dtype=torch.int32, device=self.device)[:, None]
        k, v = self.vgo.cache_read(self.cache, table, torch.zeros(pages, dtype=torch.int32, device=self.device), page, dtype=F32)
        assert torch.equal(torch.nan_to_num(k.double().cpu(), nan=1e300), torch.nan_to_num(self.pages.k, nan=1e300))
        assert torch.equal(torch.nan_to_num(v.double().cpu(), nan=1e300), torch.nan_to_num(self.pages.v, nan=1e300))
        if self.masses:
            assert torch.equal(self.cache.log_mass.double().cpu(), self.pages.mass)

    def fill(self, seed, gain=1.0):
        """Random tokens in every page."""
        pages, hk, page, d = self.pages.k.shape
        g = torch.Generator().manual_seed(seed)
        k, v = (torch.randn(pages, hk, page, d, generator=g) * gain for _ in range(2))
        mass = torch.randint(1, 9, (pages, page), generator=g).float().log() if self.masses else None
        self.append(k, v, torch.arange(pages, dtype=torch.int32)[:, None], torch.zeros(pages, dtype=torch.int32), log_mass=mass)

    def attend(self, q, table, lengths, counts=None, causal=False, scale=None):
        got = self.vgo.cached_attention(self.to(q), self.cache, self.to(table), self.to(lengths), self.to(counts), causal=causal,
                                        scale=scale)
        want, bound = oracle.attention(q, self.pages, table, lengths, counts, causal=causal, scale=scale, masses=self.masses)
        assert got.shape == q.shape and got.dtype == q.dtype
        off = (got.double().cpu() - want).abs()
        assert torch.isfinite(off).all()
        worst = (off - bound).max().item() if off.numel() else 0.0
        assert worst <= 0, f"off by {worst:.3e} beyond its bound, {off.max():.3e} in all"
        return got


# ----------------------------------------------------------------- append, read ----
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("starts,counts,n", [([0], None, 1), ([7], None, 1), ([3, 31], [5, 2], 5), ([0, 30, 61], [70, 0, 33], 70),
                                             ([5, 64], None, 129), ([8, 16], [24, 31], 32)])
def test_append(vgo, device, dtype, dim, starts, counts, n):
    b = len(starts)
    both = Both(vgo, device, b * 7 + 2, 3, 32, dim)
    both.fill(1)
    table, _ = layout(b, 7 * 32, 32, 2)
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(b, n, h, dim, generator=g).to(dtype).transpose(1, 2) for h in (3, 3, 6))
    got = both.append(k, v, table, int32(starts), None if counts is None else int32(counts), q=q, rope=tables(90, dim))
    assert got.stride(2) > got.stride(1)  # token-major, as q
    both.check_everything()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page", [32, 64, 256, 1024])
def test_append_positions_masses_and_no_rotation(vgo, device, dtype, page):
    b, n, dim = 2, 41, 64
    both = Both(vgo, device, 9, 2, page, dim, masses=True)
    both.fill(1)
    table, _ = layout(b, 3 * page, page, 2)
    g = torch.Generator().manual_seed(4)
    k, v, q = (torch.randn(b, h, n, dim, generator=g).to(dtype) for h in (2, 2, 2))
    positions = torch.randint(-2, 40, (b, n), generator=g).int()
    mass = torch.randn(b, n, generator=g)
    mass[0, 3] = -math.inf
    both.append(k, v, table, int32([page - 11, 2 * page - 5]), int32([41, 30]), q=q, rope=tables(37, dim), positions=positions,
                log_mass=mass)
    both.append(v, k, table, int32([0, 5]), int32([2, 3]))  # masses of zero
    both.check_everything()


def test_append_values_next_to_a_border(vgo, device):
    """Exact ties, their neighbours, zeros, blocks that are tiny, huge, infinite or NaN."""
    dim = 64
    both = Both(vgo, device, 2, 1, 64, dim)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], dtype=F32)
    rows = [torch.cat([ties, torch.nextafter(ties, ties * 2), torch.nextafter(ties, ties * 0), -ties]).repeat(2) * s
            for s in (1.0, 2.0 ** -20, 2.0 ** 100, 2.0 ** -126)]
    rows += [torch.zeros(64), torch.full((64,), 3.4028234663852886e38), torch.full((64,), 1e-45), torch.full((64,), -3e38)]
    bad = torch.ones(2, 64)
    bad[0, 5], bad[1, 63] = math.nan, -math.inf
    x = torch.cat([torch.stack(rows), bad])[None, None]
    both.append(x, x.flip(2), int32([[0]]), int32([3]))
    both.check_everything()
    both.append(x, x.flip(2), int32([[1]]), int32([3]), rope=tables(1, dim), positions=torch.zeros(1, x.shape[2], dtype=torch.int32))
    # (sin 0, cos 1: a rotation by nothing keeps ties ties; of the block with an infinity its partner's becomes NaN)
    pages = both.pages
    k, _ = vgo.cache_read(both.cache, both.to(int32([[1]])), both.to(int32([3])), x.shape[2], dtype=F32)
    assert torch.equal(torch.nan_to_num(k[0, 0].double().cpu(), nan=1e300), torch.nan_to_num(pages.k[1, 0, 3:3 + x.shape[2]], nan=1e300))


@pytest.mark.parametrize("case", ["no page", "past the table", "page of another cache", "before the first", "counts out of range"])
def test_tokens_without_a_place_are_left_out(vgo, device, case):
    both = Both(vgo, device, 4, 2, 32, 64, masses=True)
    both.fill(5)
    g = torch.Generator().manual_seed(6)
    k, v = torch.randn(2, 2, 40, 64, generator=g), torch.randn(2, 2, 40, 64, generator=g)
    table, starts, counts = int32([[0, 1], [2, 3]]), int32([10, 20]), None
    if case == "no page":
        table = int32([[0, -1], [-7, 3]])
    elif case == "past the table":
        starts = int32([50, 2000000000])
    elif case == "page of another cache":
        table = int32([[0, 4], [2147483647, 3]])
    elif case == "before the first":
        starts = int32([-13, -2147483648])
    else:
        counts = int32([-3, 1000])
    both.append(k, v, table, starts, counts, q=k, rope=tables(64, 64))
    both.check_everything()


def test_read_ranges(vgo, device):
    both = Both(vgo, device, 8, 2, 64, 128)
    both.fill(7)
    table = int32([[5, 1, -1], [0, 9, 3]])
    for starts, n, counts in (([3, 62], 70, None), ([0, 127], 9, [4, 9]), ([100, -4], 100, [100, 50]), ([0, 0], 1, [0, 1])):
        k, v = vgo.cache_read(both.cache, both.to(table), both.to(int32(starts)), n, None if counts is None else both.to(int32(counts)),
                              dtype=F32)
        want = oracle.read(both.pages, table, int32(starts), n, counts)
        assert torch.equal(k.double().cpu(), want[0]) and torch.equal(v.double().cpu(), want[1])
        half = vgo.cache_read(both.cache, both.to(table), both.to(int32(starts)), n, None if counts is None else both.to(int32(counts)))
        assert half[0].dtype == BF16 and torch.equal(half[0].float(), k) and torch.equal(half[1].float(), v)


# -------------------------------------------------------------------- attention ----
SHAPES = [  # batch, heads, key heads, dim, queries, tokens, page
    (1, 1, 1, 64, 1, 1, 32), (1, 4, 1, 64, 1, 33, 32), (2, 4, 4, 128, 1, 300, 64), (3, 16, 2, 64, 1, 517, 128),
    (2, 8, 2, 64, 4, 259, 64), (1, 2, 2, 128, 17, 100, 32), (1, 2, 1, 64, 50, 261, 64), (2, 6, 2, 64, 130, 333, 256),
    (1, 4, 2, 128, 150, 700, 64), (1, 1, 1, 64, 300, 300, 1024)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(vgo, device, shape, causal, dtype):
    b, h, hk, dim, n, tokens, page = shape
    table, pages = layout(b, tokens, page, 8)
    both = Both(vgo, device, pages, hk, page, dim, masses=n % 2 == 1)
    both.fill(9)
    g = torch.Generator().manual_seed(10)
    q = (torch.randn(b, n, h, dim, generator=g) * 2).to(dtype).transpose(1, 2)
    out = both.attend(q, table, torch.full((b,), tokens, dtype=torch.int32), causal=causal)
    assert h == 1 or n == 1 or out.stride(2) > out.stride(1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 3, 40, 140])
@pytest.mark.parametrize("causal", [False, True])
def test_ragged(vgo, device, dtype, n, causal):
    """Lengths of nothing, one, within and past the table; counts of nothing and all; lengths below the counts."""
    b, page = 7, 64
    table, pages = layout(b, 5 * page, page, 11)
    both = Both(vgo, device, pages, 2, page, 64, masses=True)
    both.fill(12)
    q = torch.randn(b, 4, n, 64, generator=torch.Generator().manual_seed(13)).to(dtype)
    lengths = int32([0, 1, 64, 65, 320, 1000, 200])
    counts = int32([n, n, 0, max(1, n // 2), n, n, n + 5])
    both.attend(q, table, lengths, counts, causal)


@pytest.mark.parametrize("n", [1, 40, 140])
@pytest.mark.parametrize("causal", [False, True])
def test_missing_pages_and_masses_that_leave_nothing(vgo, device, n, causal):
    page = 32
    table = int32([[0, -1, 2, 3, 99, 5], [-1, -1, -1, -1, -1, -1], [6, 7, 8, 9, 10, 11], [6, 0, 8, 2, 10, 11]])
    both = Both(vgo, device, 12, 2, page, 64, masses=True)
    both.fill(14)
    for place in ((6, slice(None)), (8, slice(5, 9)), (10, 0), (3, slice(None))):  # (a mass of -inf keeps a token out)
        both.pages.mass[place] = -math.inf
        both.cache.log_mass[place] = -math.inf
    both.pages.mass[11, 3] = both.cache.log_mass[11, 3] = torch.finfo(F32).min
    q = torch.randn(4, 2, n, 64, generator=torch.Generator().manual_seed(15))
    both.attend(q, table, int32([190, 192, 170, 32]), causal=causal)


@pytest.mark.parametrize("n", [1, 40, 140])
def test_masked_places_may_hold_anything(vgo, device, n):
    """Tokens past the length: NaN blocks and masses, in the last tile and in pages beyond."""
    table, pages = layout(2, 192, 64, 16)
    both = Both(vgo, device, pages, 2, 64, 64, masses=True)
    both.fill(17)
    lengths = int32([75, 128])
    for b in range(2):
        for t in range(int(lengths[b]), 192):
            page, slot = int(table[b, t // 64]), t % 64
            bad = torch.full((1, 2, 1, 64), math.nan)
            both.append(bad, bad, int32([[page]]), int32([slot]), log_mass=torch.full((1, 1), math.nan))
            both.pages.k[page, :, slot] = both.pages.v[page, :, slot] = 0.0
            both.pages.mass[page, slot] = 0.0
    q = torch.randn(2, 4, n, 64, generator=torch.Generator().manual_seed(18))
    both.attend(q, table, lengths)
    if n > 1:
        both.attend(q, table, lengths, causal=True)


@pytest.mark.parametrize("n", [1, 140])
def test_large_equal_scores_and_large_scales(vgo, device, n):
    """Scores far from zero and far apart, one key's probability all of it."""
    table, pages = layout(1, 260, 64, 19)
    both = Both(vgo, device, pages, 1, 64, 64)
    both.fill(20, gain=8.0)
    q = torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(21)) * 8
    both.attend(q, table, int32([260]))
    both.attend(q, table, int32([260]), scale=1e-3)
    both.attend(torch.zeros(1, 2, n, 64), table, int32([260]))


def test_strides(vgo, device):
    table, pages = layout(2, 200, 64, 22)
    both = Both(vgo, device, pages, 2, 64, 64)
    both.fill(23)
    g = torch.Generator().manual_seed(24)
    wide = torch.randn(2, 9, 4, 3, 64, generator=g)
    for q in (wide[:, :, :, 1].transpose(1, 2), wide[:, ::2, :, 0].transpose(1, 2), wide[:1, :, :, 2].transpose(1, 2).expand(2, 4, 9, 64),
              torch.randn(2, 4, 64, 9, generator=g).transpose(2, 3), torch.randn(2, 4, 9, 65, generator=g)[..., 1:]):
        both.attend(q, table, int32([200, 123]))


def test_results_are_the_same_bits(vgo, device):
    table, pages = layout(2, 3000, 64, 25)
    both = Both(vgo, device, pages, 2, 64, 64)
    both.fill(26)
    for n in (1, 70, 200):
        q = torch.randn(2, 8, n, 64, generator=torch.Generator().manual_seed(27)).to(BF16).to(device)
        call = lambda: vgo.cached_attention(q, both.cache, both.to(table), both.to(int32([3000, 1234])), causal=True)
        first = call()
        for _ in range(4):
            assert torch.equal(first, call())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("what", ["small", "zeros", "keys too small", "keys too large", "values too large", "past the length"])
def test_scales_beyond_f16(vgo, device, what, causal, dim):
    """Keys and values that f16 holds, and those it does not (f16 queries, many of them: the products' type goes by it)."""
    table, pages = layout(1, 260, 64, 28)
    both = Both(vgo, device, pages, 1, 64, dim)
    both.fill(29)
    g = torch.Generator().manual_seed(30)
    scale = {"small": 2.0 ** -20, "zeros": 0.0, "keys too small": 2.0 ** -23, "keys too large": 2.0 ** 16}.get(what, 1.0)
    k, v = torch.randn(1, 1, 3, dim, generator=g) * scale, torch.randn(1, 1, 3, dim, generator=g)
    q = torch.randn(1, 2, 140, dim, generator=g).half() * (1.0 if scale <= 1 else 2.0 ** -14)
    if what == "values too large":
        v[:, :, 1] *= 2.0 ** 16
        v[:, :, 1, ::2] = 0.0
        k[:, :, 1], q = -8.0, q.abs() + 1.0  # (an improbable key: what comes out is finite in f16)
    both.append(k, v, table, int32([258 if what == "past the length" else 77]))
    if what == "past the length":
        bad = torch.full((1, 1, 2, dim), math.nan)
        both.append(bad, bad, table, int32([258]))
    both.attend(q, table, int32([258 if what == "past the length" else 260]), causal=causal)


def test_f16_probabilities_keep_their_bits(vgo, device):
    """One key far above 250 equal ones, whose probabilities are 2^-18 of it each."""
    table, pages = layout(1, 256, 64, 31)
    both = Both(vgo, device, pages, 1, 64, 64)
    k = torch.zeros(1, 1, 256, 64)
    k[0, 0, 100, 0] = 6.0
    v = torch.randn(1, 1, 256, 64, generator=torch.Generator().manual_seed(32))
    v[0, 0, 100] = 0.0
    both.append(k, v, table, int32([0]))
    q = torch.zeros(1, 1, 130, 64).half()
    q[..., 0] = 18 * math.log(2.0) / 6.0
    both.attend(q, table, int32([256]), scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
@pytest.mark.parametrize("lowest", [torch.finfo(F32).min, -1e9, -1e4])
def test_masses_of_the_lowest_value_are_numbers(vgo, device, n, dtype, lowest):
    """A sequence that has nothing else, one that has one other key, one whose first 64 keys are such."""
    table = int32([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    both = Both(vgo, device, 9, 2, 64, 64, masses=True)
    both.fill(33)
    for mass in (both.pages.mass, both.cache.log_mass):
        mass[:6] = lowest
        mass[4, 9] = 0.5
        mass[6] = lowest
    q = torch.randn(3, 4, n, 64, generator=torch.Generator().manual_seed(34)).to(dtype)
    both.attend(q, table, int32([180, 192, 150]))
    both.attend(q, table, int32([180, 192, 150]), causal=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
def test_scores_of_any_size_stay_finite(vgo, device, n, dtype):
    """Scores of 1e10, of which fp32 knows no more than hundreds: finite, and within the range of the values."""
    table, pages = layout(1, 300, 64, 35)
    both = Both(vgo, device, pages, 1, 64, 64)
    both.fill(36, gain=2.0 ** 13)
    q = (torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(37)) * 2.0 ** 14).to(dtype)
    out = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(int32([300])), scale=10.0).double().cpu()
    out = out[torch.isfinite(q).all(-1)]  # (2^16 is past f16: the scores of such a query are not finite by definition)
    assert torch.isfinite(out).all() and out.abs().max() <= both.pages.v.abs().max() * (1 + 2.0 ** -7)


# (sequences, heads, key heads, queries, tokens, channels): kept tokens enough for several pieces, joined afterwards.
LONG = [(1, 2, 1, 1, 5000, 64), (3, 16, 1, 1, 2100, 128), (2, 3, 1, 7, 3333, 64), (1, 5, 5, 1, 4097, 64), (1, 4, 2, 31, 2500, 128),
        (2, 2, 1, 33, 3000, 64), (1, 3, 1, 86, 1111, 128), (1, 1, 1, 1029, 1500, 64), (1, 1, 1, 1100, 1500, 128),
        (2, 6, 2, 350, 700, 64), (1, 1, 1, 130, 4500, 64), (1, 9, 9, 4200, 300, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", LONG)
def test_long_sequences(vgo, device, shape, causal, dtype):
    b, h, hk, n, length, d = shape
    table, pages = layout(b, length, 128, 5)
    both = Both(vgo, device, pages, hk, 128, d, masses=n % 2 == 1)
    both.fill(6)
    q = torch.randn(b, h, n, d, generator=torch.Generator().manual_seed(7)).to(dtype)
    both.attend(q, table, int32([length - 701 * i if i else length for i in range(b)]), causal=causal)


@pytest.mark.parametrize("n", [1, 3, 40, 90])
@pytest.mark.parametrize("causal", [False, True])
def test_many_sequences_of_very_different_lengths(vgo, device, n, causal):
    """More sequences than a wave has lanes, three of them far longer than the others; pages in common."""
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 200, (150,), generator=g).int()
    lengths[[3, 77, 149]] = int32([2500, 1400, 3000])
    counts = torch.randint(0, n + 1, (150,), generator=g).int()
    both = Both(vgo, device, 60, 1, 64, 64)
    both.fill(9)
    table = torch.randint(0, 60, (150, 47), generator=g).int()
    q = torch.randn(150, 2, n, 64, generator=g)
    both.attend(q, table, lengths, counts, causal=causal)
    both.attend(q, table, lengths.flip(0), counts, causal=causal)
    both.attend(q, table, lengths, causal=causal)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_lengths_beyond_any_table(vgo, device, n):
    """Queries that stand past the table see all of it, those of a negative length nothing."""
    table, pages = layout(2, 700, 64, 5)
    both = Both(vgo, device, pages, 1, 64, 64)
    both.fill(6)
    q = torch.randn(2, 2, n, 64, generator=torch.Generator().manual_seed(7))
    held = 64 * table.shape[1]
    want = both.attend(q, table, int32([held + n, 0]), causal=True)
    for ends in ([2 ** 31 - 1, -2 ** 31], [2 ** 31 - 32, -5], [2 ** 30, -1]):
        assert torch.equal(want, both.to(q).new_zeros(()) + vgo.cached_attention(both.to(q), both.cache, both.to(table),
                                                                                both.to(int32(ends)), causal=True))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,place", [(1, 140), (1, 265), (3, 50), (4, 40), (4, 70)])
def test_a_later_value_beyond_f16_leaves_earlier_rows_alone(vgo, device, dim, group, place):
    """One value that f16 does not hold, of a new token in the block of 32 in which a tile of 128 or 256 causal rows ends,
    behind the last one that the tile's rows see."""
    table, pages = layout(1, 305, 64, 40)
    both = Both(vgo, device, pages, 1, 64, dim)
    both.fill(41)
    k, v = torch.full((1, 1, 1, dim), -8.0), torch.zeros(1, 1, 1, dim)
    v[..., 1::2] = 6 * 2.0 ** 14
    both.append(k, v, table, int32([place]))
    # (an improbable key: what later rows make of it is finite in f16)
    q = torch.randn(1, group, 300, dim, generator=torch.Generator().manual_seed(42)).abs().half() + 1.0
    both.attend(q, table, int32([305]), causal=True)


def test_tiny_keys_under_a_large_scale_in_f16(vgo, device):
    """Keys of 2^-62, scores of which the largest scale makes thousandths: two keys of one size and two signs, values of two signs."""
    table, pages = layout(1, 64, 64, 56)
    both = Both(vgo, device, pages, 1, 64, 128)
    k, v = torch.full((1, 1, 2, 128), 6 * 2.0 ** -63), torch.ones(1, 1, 2, 128)
    k[:, :, 1] *= -1
    v[:, :, 1] *= -1
    both.append(k, v, table, int32([0]))
    for n in (1, 140):
        both.attend(torch.full((1, 1, n, 128), 65504.0).half(), table, int32([2]), scale=1e8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_blocks_that_cancel(vgo, device, dtype, dim):
    """Rotated blocks of one channel whose two parts, some 600 each, leave a little more than 7 or 3.5, where the scale doubles: in
    fp32 the parts' roundings alone (2^-15 each) leave less."""
    n, heads, half = 160, 2, dim // 2
    g = torch.Generator().manual_seed(43)
    pool = 1 << 18
    sin, o = torch.rand(pool, generator=g) * 0.5 + 0.3, (torch.rand(pool, generator=g) * 900 + 300).to(dtype).float()
    y = torch.tensor([7.0, 3.5])[torch.arange(pool) % 2]
    x = ((y + o * sin) / 0.6).to(dtype).float()
    cos = ((y.double() * (1 + 2.0 ** -18) + o.double() * sin.double()) / x.double()).float()
    exact = x.double() * cos.double() - o.double() * sin.double()
    in_fp32 = ((x * cos).double() - o.double() * sin.double()).float()
    chosen = ((exact > y) & (in_fp32 < y * (1 - 2.0 ** -19))).nonzero().flatten()[:n * heads * half // 32].view(half // 32, heads, n)
    assert chosen.numel() == n * heads * half // 32
    k, tables_of = torch.zeros(1, heads, n, dim), (torch.zeros(n, dim), torch.ones(n, dim))
    for block in range(half // 32):
        for head in range(heads):
            at, of = 32 * block + 5 * head + 3, chosen[block, head]
            k[0, head, :, at], k[0, head, :, at + half] = x[of], o[of]
            tables_of[0][:, at], tables_of[1][:, at] = sin[of], cos[of]
    both = Both(vgo, device, 6, heads, 32, dim)
    both.append(k.to(dtype), k.to(dtype), torch.arange(6, dtype=torch.int32)[None], int32([3]), rope=tables_of,
                positions=torch.arange(n, dtype=torch.int32)[None])
    both.check_everything()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
@pytest.mark.parametrize("length", [70, 5000])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite_come_out_as_nan(vgo, device, bad, length, n, dtype):
    """One channel of one query: its row is NaN, its neighbours are as they were, and a row that sees nothing is zeros still.
    (Whole sequences, and those cut into pieces.)"""
    table, pages = layout(1, length, 64, 44)
    both = Both(vgo, device, pages, 1, 64, 64)
    both.fill(45)
    q = torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(46)).to(dtype)
    want, bound = oracle.attention(q, both.pages, table, int32([length]))
    row = n // 3
    q[0, 1, row, 13] = bad
    got = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(int32([length]))).double().cpu()
    assert torch.isnan(got[0, 1, row]).all()
    got[0, 1, row], want[0, 1, row] = 0.0, 0.0
    assert ((got - want).abs() <= bound).all()
    none = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(int32([min(row, length)])),
                                causal=True).cpu()  # (the first n - row queries stand before the first token)
    before = n - min(row, length)
    if row < before:
        assert not none[:, :, :before].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 140])
def test_an_infinite_query_whose_scores_are_all_minus_infinity(vgo, device, n, dtype):
    table, pages = layout(1, 70, 64, 44)
    both = Both(vgo, device, pages, 1, 64, 64)
    both.fill(45)
    k = torch.full((1, 1, 70, 64), -1.0)
    both.append(k, k, table, int32([0]))
    q = torch.ones(1, 1, n, 64, dtype=dtype)
    q[0, 0, 0, 0] = math.inf
    got = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(int32([70]))).cpu()
    assert torch.isnan(got[0, 0, 0]).all() and ((got[0, 0, 1:].double() + 1).abs() <= 2.0 ** -8).all()  # (others: the values' -1)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
@pytest.mark.parametrize("masses", [False, True])
@pytest.mark.parametrize("far", [14, 20])
@pytest.mark.parametrize("first", [185, 189, -184, -188])
def test_neighbouring_scores_far_from_zero_stay_finite(vgo, device, first, far, masses, n, dtype):
    """Scores that are adjacent fp32 numbers past 2^27 or 2^33, 16 or 1,024 apart, the larger one later, and one number with the
    scale.  (Keys of 2^14 are f16 numbers, those of 2^20 are not.)"""
    scale = torch.tensor(1.4426950408889634, dtype=F32)
    low = torch.tensor(first * 2.0 ** (far + 6), dtype=F32)
    assert low * scale == (low + 2.0 ** (far - 10)) * scale != low + 2.0 ** (far - 10) != low
    table, pages = layout(1, 320, 64, 47)
    both = Both(vgo, device, pages, 1, 64, 64, masses=masses)
    k, v = torch.zeros(1, 1, 320, 64), torch.randn(1, 1, 320, 64, generator=torch.Generator().manual_seed(48))
    k[..., 0] = 2.0 ** far
    k[0, 0, 100 if n > 64 else 300, 32] = 2.0 ** (far - 10)
    both.append(k, v, table, int32([0]))
    q = torch.zeros(1, 1, n, 64)
    q[..., 0], q[..., 32] = first * 64.0, 1.0
    out = vgo.cached_attention(both.to(q.to(dtype)), both.cache, both.to(table), both.to(int32([320])), scale=1.0).double().cpu()
    assert torch.isfinite(out).all() and out.abs().max() <= both.pages.v.abs().max() * (1 + 2.0 ** -7)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
@pytest.mark.parametrize("causal", [False, True])
def test_a_mass_of_minus_infinity_keeps_out_whatever_is_stored(vgo, device, causal, n, dtype):
    """Blocks of NaN at tokens that no query sees: one in a tile, a whole tile, every second one of a page, the last one."""
    table, pages = layout(2, 260, 64, 50)
    both = Both(vgo, device, pages, 2, 64, 64, masses=True)
    both.fill(51)
    bad = torch.full((1, 2, 1, 64), math.nan)
    bad[..., 32:] = 1.0  # (a block that is a number beside it)
    for t in [0, 45, *range(64, 128), *range(128, 192, 2), 259]:
        page, slot = int(table[0, t // 64]), t % 64
        both.append(bad, bad, int32([[page]]), int32([slot]), log_mass=torch.full((1, 1), -math.inf))
        both.pages.k[page, :, slot] = both.pages.v[page, :, slot] = 0.0
    q = torch.randn(2, 4, n, 64, generator=torch.Generator().manual_seed(52)).to(dtype)
    both.attend(q, table, int32([260, 230]), causal=causal)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 40, 140])
def test_a_mass_of_nan_shows(vgo, device, n, dtype):
    """Queries that see the token are NaN; those before it, and the other sequence's, are as they were."""
    table, pages = layout(2, 260, 64, 53)
    both = Both(vgo, device, pages, 1, 64, 64, masses=True)
    both.fill(54)
    lengths, t = int32([260, 230]), 260 - n // 2 - 1
    q = torch.randn(2, 2, n, 64, generator=torch.Generator().manual_seed(55)).to(dtype)
    want, bound = oracle.attention(q, both.pages, table, lengths, causal=True, masses=True)
    both.cache.log_mass[int(table[0, t // 64]), t % 64] = math.nan
    got = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(lengths), causal=True).double().cpu()
    sees = torch.arange(260 - n, 260) >= t
    assert torch.isnan(got[0, :, sees]).all()
    got[0, :, sees], want[0, :, sees] = 0.0, 0.0
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [1, 40])
def test_few_queries_take_probabilities_to_two_terms(vgo, device, n, dtype):
    """Two keys whose values nearly cancel: what is left shows how far a probability was rounded.  A probability is the sum of two
    bf16 numbers, off by half a step, 2^-8, of half a step at most: 2^-16."""
    table, pages = layout(1, 64, 64, 57)
    both = Both(vgo, device, pages, 1, 64, 64)
    k, v = torch.zeros(1, 1, 2, 64), torch.ones(1, 1, 2, 64)
    k[0, 0, 0, 0], v[0, 0, 1] = 1.0, -2.0
    both.append(k, v, table, int32([0]))
    q = torch.zeros(1, 1, n, 64)
    q[..., 0] = 0.6796875 + torch.arange(n) * 2.0 ** -8  # (about log 2: the first key twice as probable)
    q = q.to(dtype)
    want, bound = oracle.attention(q, both.pages, table, int32([2]), scale=1.0, p_bits=2.0 ** -16)
    got = vgo.cached_attention(both.to(q), both.cache, both.to(table), both.to(int32([2])), scale=1.0).double().cpu()
    assert ((got - want).abs() <= bound).all()


def test_read_in_f16_rounds_to_nearest(vgo, device):
    """Numbers that f16 holds, those below its normal and its smallest ones, and those past it."""
    both = Both(vgo, device, 4, 2, 64, 64)
    for page, gain in enumerate((1.0, 2.0 ** -16, 2.0 ** -24, 2.0 ** 15)):
        x = torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(58 + page)) * gain
        both.append(x, x.flip(2), int32([[page]]), int32([0]))
    table, zero = both.to(int32([[0, 1, 2, 3]])), both.to(int32([0]))
    whole, half = (vgo.cache_read(both.cache, table, zero, 256, dtype=t) for t in (F32, F16))
    for x, y in zip(whole, half):
        assert y.dtype == F16 and torch.equal(x.cpu().to(F16), y.cpu()) and torch.isinf(y).any()
