"""sample_filtered at the borders between two entries: coins and top-p values on
either side of a running mass, close to it.  The definition is formed with 64-bit
mantissas (numpy's long double), so that its own rounding, 2^-64 an operation, stays far
below the distances tested.

Ids and counts are compared exactly.  That is a demand on the kernel only where a
border is farther away than the kernel's sums are off: 2^-43 of the row's mass.  The
coins of these rows are multiples of 2^-24, and `far_enough` leaves out those that lie
closer than that to a border.
"""
import numpy as np
import pytest
import torch

from test_filtered_sample import call, check

LD = np.longdouble


class Row:
    """The order, running masses and mass of one row without NaN or infinities above."""

    def __init__(self, x, T):
        x = np.asarray(x, LD)
        order = np.argsort(-x, kind="stable")
        self.order = order[x[order] > -np.inf]
        v = x[self.order]
        with np.errstate(over="ignore", under="ignore"):
            w = np.exp((v - v[0]) / LD(T))
        self.cum = np.cumsum(w)
        self.mass = self.cum[-1]

    def far_enough(self, part, share=2.0 ** -43):
        """part * mass is farther than `share` of the mass from every running mass."""
        at = np.searchsorted(self.cum, LD(part) * self.mass)
        near = self.cum[max(at - 1, 0):at + 2]
        return bool((np.abs(near - LD(part) * self.mass) > LD(share) * self.mass).all())

    def place(self, part):
        """Entries whose running mass is at most part * mass."""
        return int(np.searchsorted(self.cum, LD(part) * self.mass, side="right"))


def heads_above_a_floor(V, first, T, bits, seed, n=20):
    """Noise, and n entries some `bits` octaves of weight above it, at places from `first` on."""
    g = np.random.default_rng(seed)
    x = g.standard_normal(V)
    at = g.choice(np.arange(first, V), n, replace=False)
    x[at] = bits * np.log(2.0) * T + 0.6 * T * g.standard_normal(n)
    return x.astype(np.float32)


STEPS = (-24, -12, -6, -3, -1, 0, 1, 2, 4, 7, 13, 25)


def coins_at_borders(row, lowest=0.2):
    """Multiples of 2^-24 on either side of every border above `lowest`."""
    out = []
    for b in (row.cum / row.mass)[:40]:
        if b < lowest or b > 1 - LD(2) ** -20:
            continue
        for s in STEPS:
            c = (int(np.floor(b * 2 ** 24)) + s) / 2.0 ** 24
            if 0 <= c < 1 and row.far_enough(c):
                out.append(c)
    return np.array(out, np.float32)


def parts_at_borders(row, lowest=0.2):
    """fp32 numbers on either side of every border above `lowest`."""
    out = []
    for b in (row.cum / row.mass)[:40]:
        if b < lowest or b > 1 - LD(2) ** -20:
            continue
        near = np.float32(b)
        for s in STEPS:
            c = np.float32(near + s * np.spacing(near))
            if 0 < c < 1 and row.far_enough(c):
                out.append(c)
    return np.array(out, np.float32)


def check_borders(pkg, xs, T, dtype=torch.float32, most=4096, bits=None):
    """Every row of xs once for each coin, and once for each top-p value, at its borders, in calls of at most `most` rows."""
    logits, coins, ids, parts, kept = [], [], [], [], []
    xs = torch.from_numpy(np.stack(xs)).to(dtype)
    for i, x in enumerate(xs.float().numpy()):
        row = Row(x, np.float32(T))
        c, p = coins_at_borders(row), parts_at_borders(row)
        coins.append(c)
        parts.append(p)
        ids.append([row.order[row.place(v)] for v in c])
        kept.append([row.place(v) + 1 for v in p])
    for which, values, want in (("coin", coins, ids), ("top-p", parts, kept)):
        of = torch.from_numpy(np.repeat(np.arange(len(xs)), [len(v) for v in values]))
        values, want = np.concatenate(values), np.concatenate(want)
        assert len(values) > 0
        for lo in range(0, len(values), most):
            part = slice(lo, lo + most)
            logits = xs[of[part]].cuda()
            if which == "coin":
                got = call(pkg, logits, T, 0, 1.0, 0.0, values[part])[0]
            else:
                got = call(pkg, logits, T, 0, values[part], 0.0, np.zeros(len(values[part]), np.float32))[2]
            bad = np.nonzero(got != want[part])[0]
            assert len(bad) == 0, (f"{which}: {len(bad)} of {len(got)} rows, the first at {values[part][bad[0]]!r}: "
                                   f"{got[bad[0]]}, not {want[part][bad[0]]}")


# V and rows a call: 1024 threads a row, 256 and 128
FORMS = [(32000, 256), (32000, 4096), (8000, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0.5, 0.6, 0.7, 0.8])
@pytest.mark.parametrize("V,most", FORMS)
def test_borders_of_entries_far_above_their_warps_first(pkg, V, most, T):
    """The heads lie where each warp has read a batch of the floor before, 30 to 55 octaves below them."""
    first = 16384 if most < 297 else 4096
    xs = [heads_above_a_floor(V, first, T, bits, 100 * i + bits) for i in range(2) for bits in (30, 41, 55)]
    check_borders(pkg, xs, T, most=most)


def close_coin(rows, T, lowest, highest):
    """Of rows of logits, the ones with a coin that lies between `lowest` and `highest` of the mass from a border of
    its row; [(row, coin, id)]."""
    out = []
    for x in rows:
        row = Row(x, np.float32(T))
        share = row.cum / row.mass
        near = np.rint(share * 2 ** 24)
        away = np.abs(near / LD(2) ** 24 - share)
        for i in np.nonzero((away > lowest) & (away < highest) & (near > 0) & (near < 2 ** 24))[0]:
            c = float(near[i]) / 2.0 ** 24
            out.append((x, c, row.order[row.place(c)]))
    return out


def check_close(pkg, cases, T, dtype=torch.float32):
    x = torch.from_numpy(np.stack([c[0] for c in cases])).to(dtype).cuda()
    got = call(pkg, x, T, 0, 1.0, 0.0, np.array([c[1] for c in cases], np.float32))[0]
    bad = np.nonzero(got != np.array([c[2] for c in cases]))[0]
    assert len(bad) == 0, f"{len(bad)} of {len(got)} rows"


@pytest.mark.gpu
@pytest.mark.parametrize("T,top", [(1e-3, 60.3), (1e-3, -35.7), (1e-4, 20.6), (1e-2, 1500.3)])
def test_borders_far_from_zero_against_the_temperature(pkg, T, top):
    """Two or three entries share the mass, top / T is 3.5e4 to 2e5, and the coin is 2^-43 to 2^-39 of the mass off a
    border: fp32 sums leave it open, and what settles it has to hold the weights to 2^-43."""
    g = np.random.default_rng(int(abs(top)))
    base = (top - 100.0 + np.abs(g.standard_normal(2000))).astype(np.float32)
    step = abs(float(np.spacing(np.float32(top))))
    reach = max(int(2.0 * T / step), 40)
    heads = []
    want = LD(2) ** 24
    while len(heads) < 24:  # the first border is 1 / S of the mass: it has to fall next to a multiple of 2^-24
        near = np.float32(top) - step * g.integers(1, reach, (200000, 3)).astype(np.float64)
        w = np.exp((near.astype(np.float32).astype(LD) - LD(np.float32(top))) / LD(np.float32(T))).sum(1) + 1
        share = 1 / w
        away = np.abs(np.rint(share * want) / want - share)
        heads += [near[i] for i in np.nonzero((away > LD(2) ** -42.5) & (away < LD(2) ** -39))[0]]
    rows = []
    for h in heads[:24]:
        x = base.copy()
        x[[100, 700, 1300, 1900]] = np.concatenate([[top], h])
        rows.append(x)
    cases = close_coin(rows, T, LD(2) ** -42.5, LD(2) ** -39)
    assert len(cases) >= 24
    check_close(pkg, cases, T)


@pytest.mark.gpu
def test_borders_of_flat_rows_far_from_zero(pkg):
    """The same where no list holds the mass: a row of 32000 near 60 at T = 0.001 has a coin within 2^-40 of a border or
    two."""
    g = np.random.default_rng(5)
    rows = [(60.3 + 0.002 * g.standard_normal(32000)).astype(np.float32) for _ in range(24)]
    cases = close_coin(rows, 1e-3, LD(2) ** -42.5, LD(2) ** -39)
    assert len(cases) >= 24
    check_close(pkg, cases, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1e5, 1e30, 2e36, 1e37, 1.2e38, 3e38, float("inf")])
def test_large_temperatures_over_the_whole_range_of_logits(pkg, dtype, T):
    """Temperatures at which logits of the type's lowest value have a share; all finite logits have the same at infinity."""
    low = float(torch.finfo(dtype).min)
    for V in (2000, 40000):
        g = torch.Generator().manual_seed(V)
        x = torch.full((7, V), low)
        x[0, V // 3] = 0.0
        x[1] = torch.rand(V, generator=g) * low
        x[2, ::2] = torch.randn(V // 2, generator=g)
        x[3, V // 2:] = -float("inf")
        x[4] = (2.0 * torch.rand(V, generator=g) - 1.0) * (-low)
        x[5, ::3] = -float("inf")
        x[5, 1] = 30.0
        x[6] = torch.randn(V, generator=g)
        x = x.to(dtype).cuda()
        for k, p, q in ((0, 1.0, 0.0), (0, 0.9, 0.0), (0, 0.3, 0.0), (0, 1.0, 0.4), (50, 1.0, 0.0), (700, 0.8, 0.1)):
            for c in (0.0, 0.25, 0.5, 0.7531, 1.0):
                check(pkg, x, T, k, p, q, np.full(7, c, np.float32))


@pytest.mark.gpu
def test_infinite_logits_and_temperature(pkg):
    """Entries of +infinity share the whole mass at every temperature, an infinite one included."""
    x = torch.randn(4, 3000)
    x[:, [5, 77, 2000]] = float("inf")
    x[2, 9] = float("nan")
    x[3, 100:200] = -float("inf")
    got = call(pkg, x.cuda(), float("inf"), 0, 1.0, 0.0, np.array([0.1, 0.5, 0.9, 0.999], np.float32))
    assert got[0].tolist() == [5, 77, 2000, 2000]
    assert np.allclose(got[1], -np.log(3.0), rtol=0, atol=2.0 ** -17)
    got = call(pkg, x.cuda(), float("inf"), 0, 1.0, 0.5, np.zeros(4, np.float32))
    assert got[2].tolist() == [3] * 4


def time_of(pkg, x, rule, coins):
    """Microseconds of a call, the least of several runs of ten."""
    ids = torch.empty(x.shape[0], dtype=torch.int32, device="cuda")
    best = float("inf")
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        for _ in range(10):
            pkg.sample_filtered(x, *rule, coins=coins, out_ids=ids)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 100)
    return best


MASKS = {"first half": slice(0, 16000), "a third": slice(10000, 20000), "padding": slice(31800, 32000)}


@pytest.mark.gpu
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rule", [(0.8, 0, 0.9, 0.0), (0.8, 0, 1.0, 0.0), (0.8, 0, 1.0, 0.05), (0.8, 50, 1.0, 0.0),
                                  (0.8, 50, 0.9, 0.0), (0.8, 300, 0.95, 0.0)])
def test_masks_of_the_lowest_value_do_not_take_the_radix_path(pkg, rule, dtype, mask):
    """A masked stretch of the row, by the type's lowest value, by -10000 and by -infinity: ids as defined, and no more
    than three times the time (the radix path takes 8 to 20 times as long)."""
    x = torch.from_numpy(np.stack([heads_above_a_floor(32000, 0, 1.0, 14, s) for s in range(4)]))
    coins = np.array([0.1, 0.4, 0.6, 0.95], np.float32)
    c = torch.from_numpy(coins).cuda()
    times = []
    for value in (-float("inf"), float(torch.finfo(dtype).min), -1e4):
        y = x.clone()
        y[:, MASKS[mask]] = value
        y = y.to(dtype).cuda()
        check(pkg, y, *rule, coins)
        times.append(time_of(pkg, y, rule, c))
    assert max(times[1:]) <= 3.0 * times[0], times


@pytest.mark.gpu
@pytest.mark.parametrize("B,V", [(3, 32000), (400, 32000), (400, 5000), (3, 200003)])
def test_finite_masks_of_every_extent(pkg, B, V):
    """From one masked entry to all but one, in stretches and scattered, with top-k below and above the number of others:
    what is finite is a candidate."""
    for i, (value, dtype) in enumerate([(-1e4, torch.float16), (float(np.finfo(np.float32).min), torch.float32),
                                        (-300.0, torch.bfloat16), (-3e38, torch.bfloat16)]):
        g = np.random.default_rng(V + i)
        x = torch.from_numpy(np.stack([heads_above_a_floor(V, 0, 1.0, 12, 10 * i + s) for s in range(3)] * (B // 3 + 1))[:B])
        for left in (1, 30, 700, V // 2, V - 200, V - 1):
            at = np.sort(g.choice(V, left, replace=False)) if left % 4 else np.arange(left)
            y = torch.full_like(x, value)
            y[:, at] = x[:, at]
            y = y.to(dtype)
            rows = slice(0, 3)
            for k, p, q in ((50, 1.0, 0.0), (500, 0.9, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.0), (60, 1.0, 1e-3)):
                coins = g.integers(0, 1 << 24, B).astype(np.float32) / np.float32(1 << 24)
                if B == 3:
                    check(pkg, y.cuda(), 0.8, k, p, q, coins)
                else:  # the first rows against the definition, the others as in a call of their own
                    got = call(pkg, y.cuda(), 0.8, k, p, q, coins)
                    few = call(pkg, y[rows].cuda(), 0.8, k, p, q, coins[rows])
                    check(pkg, y[rows].cuda(), 0.8, k, p, q, coins[rows])
                    for a, b in zip(got, few):
                        assert np.array_equal(a[rows], b)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0.7, 50.0, 1e20, 3e38, float("inf")])
def test_min_p_is_the_same_with_and_without_a_nan(pkg, T):
    """A NaN sends its row another way, on which the same entries pass min-p: those of real weights, of which 1 - 1e-19
    is below a min-p of 1."""
    g = np.random.default_rng(8)
    V = 3000
    x = torch.from_numpy(g.standard_normal((6, V)).astype(np.float32))
    x[1, 40:90] = x[1].max()
    y = torch.cat([x, torch.full((6, 1), float("nan"))], 1)
    for q in (1.0, 0.999, 0.3, 7.0, 1e-30):
        a = call(pkg, x.cuda(), T, 0, 1.0, q, np.full(6, 0.5, np.float32))
        b = call(pkg, y.cuda(), T, 0, 1.0, q, np.full(6, 0.5, np.float32))
        assert a[0].tolist() == b[0].tolist() and a[2].tolist() == b[2].tolist()
        if T < 1e30 and q >= 1.0:
            assert a[2].tolist() == (x == x.amax(1, keepdim=True)).sum(1).tolist()


def rows_of_many_ties(n):
    """Rows that take the radix path: fp16 logits around 100 in steps of 1/16, hundreds of equal ones at a crossing."""
    g = np.random.default_rng(12)
    return [torch.from_numpy(100.0 + 2.9 * g.standard_normal(57481)).half().float().numpy() for _ in range(n)]


@pytest.mark.gpu
def test_last_coins_over_many_ties(pkg):
    """The largest coins fall among the lightest entries, each 2^-35 of the mass or less: sums in units that the largest
    weight sets, not the mass, count 50000 roundings there."""
    rows = rows_of_many_ties(16)
    T = 0.75
    logits, coins, ids = [], [], []
    for x in rows:
        row = Row(x, np.float32(T))
        for j in range(1, 7):
            c = 1.0 - j * 2.0 ** -24
            if row.far_enough(c):
                logits.append(x)
                coins.append(c)
                ids.append(row.order[row.place(c)])
    assert len(ids) > 80
    got = call(pkg, torch.from_numpy(np.stack(logits)).half().cuda(), T, 0, 1.0, 0.0, np.array(coins, np.float32))[0]
    assert got.tolist() == ids


@pytest.mark.gpu
def test_finite_masks_with_top_k_and_min_p(pkg):
    """Min-p leaves fewer than top-k asks for, above a masked half: the list of min-p's entries decides, as with
    -infinity."""
    x = torch.from_numpy(np.stack([heads_above_a_floor(32000, 0, 1.0, 14, s, n=300) for s in range(4)]))
    coins = np.array([0.1, 0.4, 0.6, 0.95], np.float32)
    c = torch.from_numpy(coins).cuda()
    times = []
    for value in (-float("inf"), float(np.finfo(np.float32).min)):
        y = x.clone()
        y[:, :16000] = value
        y = y.cuda()
        check(pkg, y, 0.8, 700, 1.0, 0.01, coins)
        times.append(time_of(pkg, y, (0.8, 700, 1.0, 0.01), c))
    assert times[1] <= 3.0 * times[0], times


@pytest.mark.gpu
@pytest.mark.parametrize("T,top", [(0.6, 0.0), (0.8, 40.0), (1.3, -300.0), (1e-2, 1500.3), (1e-5, 812.7), (1e-6, 90000.0)])
def test_log_probabilities_of_open_rows(pkg, T, top):
    """ln of the share of an entry of the whole row: the mass within 2^-18, whatever the logits' distance from 0 is
    against the temperature, and half a step of fp32 for the result."""
    for V in (300, 32000, 100003):
        rows = [np.float32(top) + heads_above_a_floor(V, V // 2, T, bits, bits) * np.float32(T if T < 0.1 else 1.0)
                for bits in (3, 20, 41)]
        coins = np.array([0.3, 0.6, 0.999], np.float32)
        got = call(pkg, torch.from_numpy(np.stack(rows)).cuda(), T, 0, 1.0, 0.0, coins)
        for x, i, lp in zip(rows, got[0], got[1]):
            row = Row(x, np.float32(T))
            want = (LD(x[i]) - LD(x.max())) / LD(np.float32(T)) - np.log(row.mass)
            assert abs(LD(lp) - want) <= LD(2) ** -18 + LD(2) ** -24 * abs(want), (V, float(lp), float(want))
