"""sample_filtered: temperature, top-k, top-p and min-p with one coin per row,
against the definition in 64 bits (a stable sort and a walk, numpy).

Ids, counts and flags are compared exactly: the definition's borders are hit
only by inputs made to hit them, whose weights are exact in both.  Log
probabilities are one rounding to fp32 (half a step, 2^-24 relative) of a
64-bit value; the mass in it may hold fp32 weights, off by less than
(2.1 * 48 + 20) * 2^-24 < 2^-17 relative: the argument of 2^x is rounded three
times at most (3 ln 2 of a step per bit, and weights below 2^-48 do not count),
2^x is within 2^-22, sums are trees of 5 levels joined in fp64.
"""
import ctypes

import numpy as np
import pytest
import torch

FMIN = float(np.finfo(np.float32).min)
LAST_COIN = 1.0 - 2.0 ** -24
NAN_FLAG, NONE_FLAG = 1, 2


def reference_row(x, T, k, p, q, coin):
    """id, log probability, kept count and flags of one row (float32 values)."""
    x = np.asarray(x, np.float64)
    flags = NAN_FLAG if np.isnan(x).any() else 0
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return 0, -np.inf, 0, flags | NONE_FLAG
    if not T >= np.float32(1e-6):
        return int(order[0]), 0.0, 1, flags
    v = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / float(T)))
    n = len(order)
    if q > 0:
        n = int((w >= min(float(q), 1.0)).sum())
    if k > 0:
        n = min(n, int(k))
    cum = np.cumsum(w)
    if 0 < p < 1:
        n = min(n, int((cum <= float(p) * cum[n - 1]).sum()) + 1)
    c = 0.0 if np.isnan(coin) else min(max(float(coin), 0.0), LAST_COIN)
    at = min(int((cum <= c * cum[n - 1]).sum()), n - 1)
    return int(order[at]), float(np.log(w[at] / cum[n - 1])), n, flags


def reference(x, T, k, p, q, coins):
    B = len(x)
    rows = [reference_row(x[b], *(np.broadcast_to(np.asarray(s), (B,))[b] for s in (T, k, p, q, coins)))
            for b in range(B)]
    return [np.array(c) for c in zip(*rows)]


def call(pkg, logits, T, k, p, q, coins, tail=3, **kw):
    """Runs the call into buffers with `tail` rows behind the last, which have to stay as they are."""
    B = logits.shape[0]
    dev = logits.device
    ids = torch.full((B + tail,), -7, dtype=torch.int32, device=dev)
    lp = torch.full((B + tail,), 77.0, device=dev)
    kept = torch.full((B + tail,), -7, dtype=torch.int32, device=dev)
    flags = torch.full((B + tail,), -7, dtype=torch.int32, device=dev)
    args = {}
    vals = {}
    for name, v, dt in (("temperature", T, np.float32), ("topk", k, np.int32), ("topp", p, np.float32),
                        ("minp", q, np.float32)):
        if np.ndim(v):
            args[name + "_rows"] = torch.from_numpy(np.asarray(v, dt)).to(dev)
            vals[name] = 0
        else:
            vals[name] = v
    got = pkg.sample_filtered(logits, vals["temperature"], vals["topk"], vals["topp"], vals["minp"],
                              coins=None if coins is None else torch.from_numpy(np.asarray(coins, np.float32)).to(dev),
                              out_ids=ids[:B], logprobs_out=lp[:B], kept_out=kept[:B], row_flags=flags[:B],
                              **args, **kw)
    torch.cuda.synchronize()
    assert got.data_ptr() == ids.data_ptr()
    for t, v in ((ids, -7), (lp, 77.0), (kept, -7), (flags, -7)):
        assert bool((t[B:] == v).all())
    return [t[:B].cpu().numpy() for t in (ids, lp, kept, flags)]


def check(pkg, logits, T, k, p, q, coins):
    got = call(pkg, logits, T, k, p, q, coins)
    as_np = (lambda s: np.asarray(s, np.float32))
    want = reference(logits.float().cpu().numpy(), as_np(T), np.asarray(k), as_np(p), as_np(q), as_np(coins))
    for name, g, w in zip(("ids", "kept", "flags"), (got[0], got[2], got[3]), (want[0], want[2], want[3])):
        bad = np.nonzero(g != w)[0]
        assert len(bad) == 0, f"{name}: rows {bad[:5]} have {g[bad[:5]]}, not {w[bad[:5]]}"
    lp, ref = got[1].astype(np.float64), want[1]
    both = np.isfinite(ref)
    assert np.array_equal(lp[~both], ref[~both])
    lp, ref = np.where(both, lp, 0.0), np.where(both, ref, 0.0)
    assert np.all(np.abs(lp - ref) <= 2.0 ** -24 * np.abs(ref) + 2.0 ** -17)


def rows(kind, B, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    n = torch.randn(B, V, generator=g)
    if kind == "normal2":
        x = 2.0 * n
    elif kind == "normal3":
        x = 3.0 * n
    elif kind == "flat":
        x = 0.05 * n
    elif kind == "far":  # far from zero, where a 16-bit logit has coarse steps
        x = 60.0 + 4.0 * n
    else:  # a few likely tokens above a broad floor
        x = 2.2 * n + (torch.rand(B, V, generator=g) < 30.0 / V) * (12.0 + 3.0 * torch.rand(B, V, generator=g))
    return x.to(dtype)


def coins_of(B, seed):
    return (np.random.default_rng(seed).integers(0, 1 << 24, B) / float(1 << 24)).astype(np.float32)


RULES = {
    "open": (0.9, 0, 1.0, 0.0),
    "topk": (0.8, 50, 1.0, 0.0),
    "topk1": (0.8, 1, 1.0, 0.0),
    "topk_large": (1.1, 1500, 1.0, 0.0),
    "topp": (0.7, 0, 0.9, 0.0),
    "topp_low": (1.0, 0, 0.05, 0.0),
    "topp_high": (1.3, 0, 0.999, 0.0),
    "minp": (1.0, 0, 1.0, 0.05),
    "all": (0.9, 40, 0.9, 0.02),
    "all_large": (1.2, 3000, 0.97, 1e-6),
    "greedy": (0.0, 40, 0.9, 0.02),
}


@pytest.mark.gpu
@pytest.mark.parametrize("rule", sorted(RULES))
@pytest.mark.parametrize("kind", ["peaked", "normal2", "normal3", "flat", "far"])
def test_rules_and_shapes(pkg, rule, kind):
    for i, (B, V) in enumerate([(7, 32000), (3, 1000), (2, 4099)]):
        check(pkg, rows(kind, B, V, 10 * i + 1).cuda(), *RULES[rule], coins_of(B, i))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 127, 511, 513, 8191, 8193, 32767, 32769, 50021, 131072, 200003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lengths_and_types(pkg, V, dtype):
    for rule in ("open", "topp", "all"):
        check(pkg, rows("normal2", 3, V, V, dtype).cuda(), *RULES[rule], coins_of(3, V))
    check(pkg, rows("peaked", 3, V, V + 1, dtype).cuda(), *RULES["topk"], coins_of(3, V + 1))


@pytest.mark.gpu
def test_largest_vocabulary(pkg):
    V = pkg.FILTERED_MAX_VOCAB
    x = rows("normal2", 2, V, 5, torch.bfloat16).cuda()
    for rule in ("open", "topp", "all"):
        check(pkg, x, *RULES[rule], coins_of(2, 9))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2, 17, 148, 149, 600])
def test_batches_with_settings_by_row(pkg, B):
    rng = np.random.default_rng(B)
    V = 2003
    T = rng.choice([0.0, 0.3, 0.8, 1.0, 2.0, -1.0, 5e-7], B).astype(np.float32)
    k = rng.choice([0, 1, 5, 50, 500, V, 2 * V, -3], B).astype(np.int32)
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0, -1.0], B).astype(np.float32)
    q = rng.choice([0.0, 0.01, 0.3, 1.0, 3.0, -1.0], B).astype(np.float32)
    check(pkg, rows("peaked", B, V, B).cuda(), T, k, p, q, coins_of(B, B))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,pad,offset", [(32000, 1, 0), (32000, 8, 1), (1001, 0, 3), (50021, 27, 5), (4096, 4096, 2)])
def test_strides_and_alignment(pkg, dtype, V, pad, offset):
    B = 5
    buf = torch.full((offset + B * (V + pad),), float("nan"), dtype=dtype, device="cuda")  # NaN wherever no row is
    x = buf[offset:].as_strided((B, V), (V + pad, 1))
    x.copy_(rows("normal2", B, V, V + pad, dtype))
    check(pkg, x, *RULES["all_large"], coins_of(B, 3))
    check(pkg, x, *RULES["open"], coins_of(B, 4))
    check(pkg, x, *RULES["topk"], coins_of(B, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [5, 700, 40000])
def test_masks_infinities_and_nan(pkg, dtype, V):
    low = float(torch.finfo(dtype).min)
    x = rows("normal2", 14, V, 77)
    x[0] = -float("inf")                        # nothing left
    x[1] = float("nan")                         # nothing left
    x[2] = -float("inf"); x[2, V - 2] = -3.0    # one left
    x[3] = low                                  # all masked by the type's lowest value: uniform
    x[4] = low; x[4, 1] = 0.5                   # one above it
    x[5, ::2] = -float("inf")
    x[6, 1::2] = float("nan")
    x[7, V // 2] = float("inf")                 # takes everything
    x[8, [1, V - 1]] = float("inf")             # shared
    x[9] = 0.0; x[9, ::2] = -0.0                # equal: -0 and 0 are
    x[10] = float("inf")
    x[11, 3:] = low
    x[12] = -float("inf"); x[12, 0] = float("nan"); x[12, V - 1] = low
    x[13, 1:] = -float("inf"); x[13, 0] = float("inf")
    x = x.to(dtype).cuda()
    for rule in ("open", "topp", "topk", "minp", "all", "topp_low", "greedy"):
        for c in (0.0, 0.37, LAST_COIN):
            check(pkg, x, *RULES[rule], np.full(14, c, np.float32))


@pytest.mark.gpu
def test_borders_that_are_exact(pkg):
    """Equal logits have weights of exactly 1, so bounds can be met exactly: top-p keeps what exceeds it, the
    draw takes the first entry whose running mass exceeds coin * total."""
    V = 1024
    x = torch.zeros(8, V, device="cuda")
    for p, c in ((0.5, 0.0), (0.5, 0.5), (0.25, 0.75), (1.0, 0.5), (1.0, 1.0 - 2.0 ** -10), (1.0, 0.25)):
        check(pkg, x, 1.0, 0, p, 0.0, np.full(8, c, np.float32))
        check(pkg, x, 1.0, 512, p, 0.0, np.full(8, c, np.float32))
        check(pkg, x, 1.0, 0, p, 1.0, np.full(8, c, np.float32))
    got = call(pkg, x, 1.0, 0, 0.5, 0.0, np.full(8, 0.5, np.float32))
    assert got[2].tolist() == [513] * 8 and got[0].tolist() == [256] * 8


@pytest.mark.gpu
def test_ties_at_the_cut(pkg):
    """Coarse logits: hundreds of equal entries around every cut, which the lowest indices survive."""
    g = torch.Generator().manual_seed(3)
    for V in (3000, 32000, 90001):
        x = torch.randint(-8, 4, (6, V), generator=g).float().cuda()
        for rule in RULES:
            check(pkg, x, *RULES[rule], coins_of(6, V))
        check(pkg, x, 0.9, V // 3, 0.95, 0.0, coins_of(6, V + 1))
        check(pkg, x, 30.0, V // 2, 0.5, 0.0, coins_of(6, V + 2))


@pytest.mark.gpu
def test_coins_out_of_range(pkg):
    x = rows("normal2", 6, 5000, 8).cuda()
    coins = np.array([-1.0, 0.0, 1.0, 5.0, np.nan, np.inf], np.float32)
    for rule in ("open", "topp", "all"):
        check(pkg, x, *RULES[rule], coins)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.05, 50.0, 1e6, 3e38, float("inf")])
def test_temperatures(pkg, T):
    x = rows("normal3", 4, 32000, 21).cuda()
    for rule in ("open", "topp", "all_large"):
        _, k, p, q = RULES[rule]
        check(pkg, x, T, k, p, q, coins_of(4, 5))


@pytest.mark.gpu
def test_top_k_beyond_32_bits_is_off(pkg):
    x = rows("peaked", 3, 2001, 6).cuda()
    c = torch.from_numpy(coins_of(3, 2)).cuda()
    kept = torch.empty(3, dtype=torch.int32, device="cuda")
    for k in (2 ** 32 + 1, 2 ** 40, -2 ** 40):
        pkg.sample_filtered(x, 1.0, k, 1.0, 0.0, coins=c, kept_out=kept)
        assert kept.tolist() == [2001] * 3


@pytest.mark.gpu
def test_nan_settings_are_off(pkg):
    x = rows("peaked", 4, 3001, 2).cuda()
    nan = float("nan")
    a = call(pkg, x, 0.8, 0, nan, nan, coins_of(4, 1))
    b = call(pkg, x, 0.8, 0, 1.0, 0.0, coins_of(4, 1))
    g = call(pkg, x, nan, 0, 1.0, 0.0, coins_of(4, 1))
    for u, v in zip(a, b):
        assert np.array_equal(u, v)
    assert g[0].tolist() == x.argmax(1).tolist() and g[2].tolist() == [1] * 4


@pytest.mark.gpu
def test_draws_from_the_row_states(pkg, orc):
    """Without coins each row draws one from its xorshift state; greedy rows draw none."""
    B, V = 9, 4001
    x = rows("normal2", B, V, 4).cuda()
    seeds = pkg.workloads.row_seeds(B, seed=5)
    T = np.array([0.8, 0.0] * 4 + [1.0], np.float32)
    st = torch.from_numpy(seeds.view(np.int64).copy()).cuda()
    got = call(pkg, x, T, 0, 0.9, 0.0, None, rng_state=st)
    after = st.cpu().numpy().view(np.uint64)
    drawn = [orc.coin(int(s)) for s in seeds]
    want = reference(x.cpu().numpy(), T, 0, np.float32(0.9), 0.0, np.array([c for c, _ in drawn], np.float32))
    assert np.array_equal(got[0], want[0])
    for b in range(B):
        assert int(after[b]) == (int(seeds[b]) if T[b] == 0 else int(drawn[b][1]))


@pytest.mark.gpu
def test_agrees_with_the_top_p_of_sample_batched(pkg):
    """Same logits, coins and top-p as sample_batched, which rounds as the reference does: the same ids up to coins
    within fp32 rounding of a border."""
    w = pkg.workloads.topp(rows=256)
    x = torch.from_numpy(w["logits"]).cuda()
    p = torch.from_numpy(w["topp_rows"]).cuda()
    coins = torch.from_numpy(coins_of(256, 1)).cuda()
    a = pkg.sample_batched(x, w["temperature"], 0.9, topp_rows=p, coins=coins)
    b = pkg.sample_filtered(x, w["temperature"], 0, 0.9, 0.0, topp_rows=p, coins=coins)
    torch.cuda.synchronize()
    assert int((a != b).sum()) <= 2


@pytest.mark.gpu
def test_repeats_streams_and_graphs(pkg):
    """The same ids whatever runs beside the call: twice, on two streams at once, captured and replayed with other
    inputs."""
    B, V = 64, 32000
    x = rows("normal2", B, V, 6).cuda()
    y = rows("peaked", B, V, 7).cuda()
    c = torch.from_numpy(coins_of(B, 2)).cuda()
    run = lambda t, **kw: pkg.sample_filtered(t, 0.9, 0, 0.95, 0.0, coins=c, **kw)  # noqa: E731
    want_x, want_y = run(x).clone(), run(y).clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(20)]
    for i, o in enumerate(outs):
        run(x if i % 2 else y, out_ids=o, stream=s1 if i % 2 else s2)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want_x if i % 2 else want_y)
    buf, ids = x.clone(), torch.empty(B, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(buf, out_ids=ids)
    for t, want in ((y, want_y), (x, want_x)):
        buf.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, want)


@pytest.mark.gpu
def test_rows_past_two_to_the_31_elements(pkg):
    """Offsets of the last rows do not fit 32 bits."""
    B, V, ld = 5, 1000, 600_000_000
    buf = torch.empty((B - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((B, V), (ld, 1))
    x.copy_(rows("normal2", B, V, 3, torch.bfloat16))
    check(pkg, x, *RULES["all"], coins_of(B, 1))


@pytest.mark.gpu
def test_empty_batch_and_python_refusals(pkg):
    x = torch.zeros(4, 100, device="cuda")
    c = torch.zeros(4, device="cuda")
    assert pkg.sample_filtered(x[:0], 1.0, 0, 1.0, 0.0, coins=c[:0]).numel() == 0
    bad = [
        lambda: pkg.sample_filtered(x.double(), 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.sample_filtered(x.t(), 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.sample_filtered(x[0], 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.sample_filtered(x[:1].expand(4, 100), 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.sample_filtered(x.cpu(), 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c[:3]),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c.cpu()),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c.double()),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c, topk_rows=c),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c, out_ids=c),
        lambda: pkg.sample_filtered(x, 1.0, 0, 1.0, 0.0, coins=c, kept_out=torch.zeros(5, dtype=torch.int32).cuda()),
        lambda: pkg.sample_filtered(torch.zeros(1, pkg.FILTERED_MAX_VOCAB + 1, dtype=torch.float16, device="cuda"),
                                    1.0, 0, 1.0, 0.0, coins=c[:1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(pkg.SamplerError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_c_refusals_before_any_device_work(pkg):
    """The C entry point checks its arguments before it touches a device (these calls pass addresses that are
    never read)."""
    L = pkg.lib()
    cfg = lambda **kw: pkg.SamplerFilterConfig(**{**dict(vocab_size=100, logits_dtype=0, temperature=1.0, topk=0,  # noqa: E731
                                                         topp=1.0, minp=0.0), **kw})

    def rc(c, logits=4096, batch=2, ld=100, coins=4096, state=None, ids=4096):
        return L.sampler_filtered(None if c is None else ctypes.byref(c), logits, batch, ld, None, None, None, None,
                                  coins, state, ids, None, None, None, None)

    assert rc(None) == -1
    assert rc(cfg(), logits=None) == -1
    assert rc(cfg(), ids=None) == -1
    assert rc(cfg(), batch=-1) == -1
    assert rc(cfg(), ld=99) == -1
    assert rc(cfg(vocab_size=0)) == -1
    assert rc(cfg(vocab_size=pkg.FILTERED_MAX_VOCAB + 1), ld=1 << 40) == -2
    assert rc(cfg(logits_dtype=3)) == -1
    assert rc(cfg(logits_dtype=-1)) == -1
    assert rc(cfg(), coins=None) == -1
    assert rc(cfg(), logits=4097) == -1
    assert rc(cfg(logits_dtype=1), logits=4097) == -1
    assert "aligned" in L.sampler_last_error().decode()
    assert rc(cfg(), batch=0) == 0
    assert rc(cfg(temperature=0.0), coins=None, batch=0) == 0


def test_reference_walk_on_known_rows():
    """The definition this file checks against, on rows worked out by hand."""
    x = [0.0, np.log(2.0), np.log(4.0), -np.inf]          # weights 1/4, 1/2, 1 in falling order 2, 1, 0
    assert reference_row(x, 1.0, 0, 1.0, 0.0, 0.0)[:3:2] == (2, 3)
    assert reference_row(x, 1.0, 0, 1.0, 0.0, 0.6)[0] == 1
    assert reference_row(x, 1.0, 0, 1.0, 0.0, 0.9)[0] == 0
    assert reference_row(x, 1.0, 2, 1.0, 0.0, 0.9)[:3:2] == (1, 2)
    assert reference_row(x, 1.0, 0, 0.5, 0.0, 0.9)[:3:2] == (2, 1)
    assert reference_row(x, 1.0, 0, 1.0, 0.4, 0.9)[:3:2] == (1, 2)
    assert reference_row(x, 0.0, 0, 1.0, 0.0, 0.9)[:3:2] == (2, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [32000, 128000])
def test_heavy_entries_side_by_side(pkg, dtype, V):
    """Most of the mass in a few entries that lie next to one another, above a broad floor: the
    largest of a stretch says little of its mass.  Row by row another number of them, up to rows
    in which they hold just less than top-p asks for."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(12, V, generator=g) * 2.2
    for b in range(12):
        x[b, 4096:4096 + 8] = torch.linspace(18.0, 15.0 - 0.25 * b, 8)
        x[b, 9000 + 700 * b: 9000 + 700 * b + 3] = 16.0
    x = x.to(dtype).cuda()
    for p in (0.5, 0.9, 0.95, 0.99):
        check(pkg, x, 0.8, 0, p, 0.0, coins_of(12, 31))
        check(pkg, x, 1.0, 0, p, 0.0, coins_of(12, 32))
    check(pkg, x, 0.8, 0, 1.0, 0.0, coins_of(12, 33))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_of_equal_logits(pkg, dtype):
    """All weights 1, so every border is exact: ids and counts follow from integers."""
    for V in (31, 1000, 32001):
        x = torch.full((4, V), 2.5, dtype=dtype).cuda()
        x[3, V // 2] = float("nan")
        for rule in ("open", "topp", "all"):
            check(pkg, x, *RULES[rule], coins_of(4, V))
