"""The operators of the 8-bit decode step and of filtered sampling, as cases that can be measured.

Three kinds of case:

  sample    token ids from logits by temperature, top-k, top-p and min-p with one given random
            number (coin) per row: pkg.sample_filtered
  quantize  float8 e4m3 values with one fp32 scale per block of 128: pkg.quantize_fp8 (activations,
            1 x 128; weights, 128 x 128) and pkg.rmsnorm_fp8 (the final RMSNorm in the same pass)
  product   classifier logits from such operands: pkg.classifier_logits_fp8

`own` chooses between the package's kernels and the plain form in elementary torch operations.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
BLOCK = 128
SMALLEST_SCALE = 2.0 ** -126  # of a block of zeros
GREEDY_BELOW = 1e-6           # rows with a lower temperature take the argmax
EPS = 1e-5                    # of the RMSNorm
LARGEST_COIN = 1.0 - 2.0 ** -24


def listed():
    s = dict(kind="sample")
    q = dict(kind="quantize")
    p = dict(kind="product")
    return [
        # one token of one user: latency; the vocabulary of the benchmark
        dict(s, name="sample 1x32000 top-k", rows=1, vocab=32000, pad=0, dtype="fp32", shape="peaked",
             rule="topk_topp", temperature=0.8, topk=50, topp=0.9, minp=0.0, masked=0.0),
        # a serving batch over a large vocabulary, bf16 logits
        dict(s, name="sample 64x128000 top-p", rows=64, vocab=128000, pad=0, dtype="bf16", shape="peaked",
             rule="topp", temperature=1.0, topk=0, topp=0.95, minp=0.0, masked=0.0),
        # the benchmark's batch: 4096 rows, Gumbel noise with a Zipf bonus, T = 0.7
        dict(s, name="sample 4096x32000 top-p", rows=4096, vocab=32000, pad=0, dtype="fp32", shape="zipf",
             rule="topp", temperature=0.7, topk=0, topp=0.9, minp=0.0, masked=0.0),
        # nothing filtered and a flat distribution: the whole vocabulary can be drawn
        dict(s, name="sample 1024x32000 open", rows=1024, vocab=32000, pad=0, dtype="fp32", shape="normal3",
             rule="open", temperature=0.8, topk=0, topp=1.0, minp=0.0, masked=0.0),
        # odd vocabulary inside a padded buffer, every row its own settings, a tenth of it masked
        dict(s, name="sample 301x50021 mixed", rows=301, vocab=50021, pad=27, dtype="fp16", shape="peaked",
             rule="mixed", temperature=0.9, topk=40, topp=0.9, minp=0.05, masked=0.1),
        # decode: the norm of one token's hidden state
        dict(q, name="rmsnorm 1x4096", rows=1, dim=4096, dtype="fp32", form="norm"),
        # the benchmark's fused batch: 8192 hidden states
        dict(q, name="rmsnorm 8192x4096", rows=8192, dim=4096, dtype="fp32", form="norm"),
        # the classifier's weights at load time
        dict(q, name="weights 32000x4096", rows=32000, dim=4096, dtype="bf16", form="weights"),
        # one token: a stream of the weights
        dict(p, name="product 1x4096x32000", rows=1, dim=4096, vocab=32000, out="fp32"),
        # a decode batch
        dict(p, name="product 32x4096x32000", rows=32, dim=4096, vocab=32000, out="fp32"),
        # ragged in every direction
        dict(p, name="product 333x1104x50021", rows=333, dim=1104, vocab=50021, out="bf16"),
        # the benchmark's fused batch
        dict(p, name="product 8192x4096x32000", rows=8192, dim=4096, vocab=32000, out="fp32"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["sample", "quantize", "product"])
    if kind == "sample":
        vocab = log_int(500, 200000)
        rows = log_int(1, min(4096, 4096 * 32000 // vocab))
        rule = rng.choice(["topk", "topp", "minp", "topk_topp", "open", "mixed"])
        return dict(kind=kind, rows=rows, vocab=vocab, pad=rng.choice([0, 0, rng.randint(1, 64)]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    shape=rng.choice(["peaked", "zipf", "normal2", "normal3"]), rule=rule,
                    temperature=round(rng.uniform(0.5, 1.3), 3), topk=log_int(1, 2000),
                    topp=round(rng.uniform(0.5, 0.99), 3), minp=round(rng.uniform(0.01, 0.2), 3),
                    masked=rng.choice([0.0, 0.0, 0.3]))
    if kind == "quantize":
        dim = log_int(128, 8192)
        return dict(kind=kind, rows=log_int(1, min(32000, 32000 * 4096 // dim)), dim=dim,
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), form=rng.choice(["norm", "rows", "weights"]))
    dim = 16 * log_int(4, 512)
    vocab = log_int(256, min(131072, 2 * 32000 * 4096 // dim))
    rows = log_int(1, min(8192, 8192 * 4096 * 32000 // (dim * vocab)))
    return dict(kind=kind, rows=rows, dim=dim, vocab=vocab, out=rng.choice(["fp32", "bf16"]))


# ---- inputs -------------------------------------------------------------------------------

def _logits(case, g):
    B, V = case["rows"], case["vocab"]
    n = torch.randn(B, V, generator=g, device=DEV)
    if case["shape"] == "normal2":
        return n * 2.0
    if case["shape"] == "normal3":
        return n * 3.0
    u = torch.rand(B, V, generator=g, device=DEV).clamp_(1e-7, 1.0 - 1e-7)
    gumbel = -torch.log(-torch.log(u))
    if case["shape"] == "zipf":  # Gumbel noise and a bonus that falls with the token's rank, 0 to 12 nats
        rank = torch.argsort(torch.rand(B, V, generator=g, device=DEV), dim=1).float() + 1.0
        return gumbel + 12.0 * torch.rand(B, 1, generator=g, device=DEV) * rank ** -1.1
    # "peaked": as a trained model answers, a few likely tokens far above a broad floor
    head = torch.rand(B, V, generator=g, device=DEV) < 40.0 / V
    return n * 2.2 + head * (gumbel * 2.0 + 13.0)


def _block_scales(x, block_rows):
    R, D = x.shape
    pr, pd = -R % block_rows, -D % BLOCK
    a = torch.nn.functional.pad(x.abs(), (0, pd, 0, pr))
    a = a.reshape((R + pr) // block_rows, block_rows, (D + pd) // BLOCK, BLOCK)
    return (a.amax(dim=(1, 3)) / FP8_MAX).clamp(min=SMALLEST_SCALE)


def _spread(scales, R, D, block_rows):
    return scales.repeat_interleave(block_rows, 0)[:R].repeat_interleave(BLOCK, 1)[:, :D]


def _quantize(x, block_rows):
    s = _block_scales(x, block_rows)
    q = (x / _spread(s, x.shape[0], x.shape[1], block_rows)).clamp(-FP8_MAX, FP8_MAX).to(FP8)
    return q, s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = case["rows"]
    st = dict(case=case)
    if case["kind"] == "sample":
        V = case["vocab"]
        x = _logits(case, g)
        if case["masked"]:
            x = x.masked_fill(torch.rand(1, V, generator=g, device=DEV) < case["masked"], -math.inf)
        buf = torch.full((B, V + case["pad"]), math.nan, dtype=DTYPES[case["dtype"]], device=DEV)
        st["logits"] = buf[:, :V]
        st["logits"].copy_(x)
        st["coins"] = torch.randint(0, 1 << 24, (B,), generator=g, device=DEV).float() / (1 << 24)
        rule = case["rule"]
        st["topk"] = case["topk"] if rule in ("topk", "topk_topp") else 0
        st["topp"] = case["topp"] if rule in ("topp", "topk_topp") else 1.0
        st["minp"] = case["minp"] if rule == "minp" else 0.0
        st["rows"] = {}
        if rule == "mixed":  # requests of several users in one batch: each filter on or off by row
            on = torch.rand(4, B, generator=g, device=DEV)
            st["rows"] = dict(
                temperature_rows=torch.where(on[0] < 0.1, 0.0, case["temperature"] * (0.8 + 0.4 * on[0])).float(),
                topk_rows=torch.where(on[1] < 0.5, (case["topk"] * (0.5 + on[1])).int() + 1, 0).int(),
                topp_rows=torch.where(on[2] < 0.5, case["topp"], 1.0).float(),
                minp_rows=torch.where(on[3] < 0.5, case["minp"], 0.0).float())
        st["out_ids"] = torch.empty(B, dtype=torch.int32, device=DEV)
        st["logprobs_out"] = torch.empty(B, dtype=torch.float32, device=DEV)
        st["kept_out"] = torch.empty(B, dtype=torch.int32, device=DEV)
    elif case["kind"] == "quantize":
        if case["form"] == "weights":
            x = torch.randn(B, case["dim"], generator=g, device=DEV) * 0.02
        else:  # hidden states: a few channels far larger than the rest
            x = torch.randn(B, case["dim"], generator=g, device=DEV) * 3.0
            x *= 1.0 + 20.0 * (torch.rand(case["dim"], generator=g, device=DEV) < 0.01)
        st["x"] = x.to(DTYPES[case["dtype"]])
        st["norm_weight"] = 1.0 + 0.1 * torch.randn(case["dim"], generator=g, device=DEV)
        st["block_rows"] = BLOCK if case["form"] == "weights" else 1
    else:
        h = torch.randn(B, case["dim"], generator=g, device=DEV)
        w = torch.randn(case["vocab"], case["dim"], generator=g, device=DEV) * 0.02
        st["h"], st["h_scales"] = _quantize(h, 1)
        st["w"], st["w_scales"] = _quantize(w, BLOCK)
        st["logits_out"] = torch.empty(B, case["vocab"], dtype=DTYPES[case["out"]], device=DEV)
    return st


# ---- the plain forms ------------------------------------------------------------------------

def _settings(st, dtype=torch.float64):
    """temperature, top-k, top-p and min-p of every row as columns."""
    B = st["case"]["rows"]
    given = dict(temperature=st["case"]["temperature"], topk=st["topk"], topp=st["topp"], minp=st["minp"])
    cols = []
    for name, v in given.items():
        r = st["rows"].get(name + "_rows")
        col = torch.full((B,), v, dtype=torch.float32, device=DEV) if r is None else r
        cols.append(col.to(torch.int64 if name == "topk" else dtype)[:, None])
    return cols


def _plain_sample(st):
    # weights, sums and comparisons with a border in 64 bits: an id on the wrong side is another id
    T, k, p, mp = _settings(st)
    x, order = torch.sort(torch.nan_to_num(st["logits"].float(), nan=-math.inf, posinf=math.inf, neginf=-math.inf),
                          dim=1, descending=True, stable=True)
    x = x.double()
    top = x[:, :1]
    greedy = ~(T >= GREEDY_BELOW)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, T)))
    w = torch.where(x > -math.inf, w, 0.0)
    there = (x > -math.inf).sum(1, keepdim=True)
    n = torch.where((k > 0) & (k < there), k, there)
    n = torch.where(mp > 0, torch.minimum(n, (w >= mp.clamp(max=1.0)).logical_and(x > -math.inf).sum(1, keepdim=True)), n)
    n = torch.where(greedy, there.clamp(max=1), n)
    cum = torch.cumsum(w, 1)
    last = (n - 1).clamp(min=0)
    cut = (cum <= p * cum.gather(1, last)).sum(1, keepdim=True) + 1
    n = torch.where((p > 0) & (p < 1), torch.minimum(n, cut), n)
    last = (n - 1).clamp(min=0)
    total = cum.gather(1, last)
    u = st["coins"].double()[:, None].clamp(0.0, LARGEST_COIN) * total
    at = torch.minimum((cum <= u).sum(1, keepdim=True), last)
    lp = torch.log(w.gather(1, at) / total)
    none = there == 0
    ids = torch.where(none, 0, order.gather(1, at))
    lp = torch.where(none, -math.inf, lp)
    return {"ids": ids[:, 0].int(), "logprobs": lp[:, 0].float(), "kept": n[:, 0].int()}


def _plain_norm(x, weight):
    x = x.float()
    return weight * (x * (1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)))


def _plain_product(st):
    h = st["h"].float() * _spread(st["h_scales"], *st["h"].shape, 1)
    w = st["w"].float() * _spread(st["w_scales"], *st["w"].shape, BLOCK)
    return torch.matmul(h, w.t()).to(st["logits_out"].dtype)


def run(state):
    kind = state["case"]["kind"]
    if own:
        from __graft_entry__ import load_package
        pkg = load_package()
        if kind == "sample":
            ids = pkg.sample_filtered(state["logits"], state["case"]["temperature"], state["topk"], state["topp"],
                                      state["minp"], coins=state["coins"], out_ids=state["out_ids"],
                                      logprobs_out=state["logprobs_out"], kept_out=state["kept_out"],
                                      **state["rows"])
            return {"ids": ids, "logprobs": state["logprobs_out"], "kept": state["kept_out"]}
        if kind == "quantize":
            if state["case"]["form"] == "norm":
                q, s = pkg.rmsnorm_fp8(state["x"], state["norm_weight"])
            else:
                q, s = pkg.quantize_fp8(state["x"], state["block_rows"])
            return {"values": q, "scales": s}
        return {"logits": pkg.classifier_logits_fp8(state["h"], state["h_scales"], state["w"], state["w_scales"],
                                                    logits_out=state["logits_out"])}
    if kind == "sample":
        return _plain_sample(state)
    if kind == "quantize":
        x = state["x"].float()
        if state["case"]["form"] == "norm":
            x = _plain_norm(x, state["norm_weight"])
        q, s = _quantize(x, state["block_rows"])
        return {"values": q, "scales": s}
    return {"logits": _plain_product(state)}


def work(case):
    B = case["rows"]
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        settings = 16 * B if case["rule"] == "mixed" else 0
        # one subtraction, scaling, exponential and addition for each logit
        return {"bytes": B * case["vocab"] * size + settings + 16 * B, "flops": 4 * B * case["vocab"]}
    if case["kind"] == "quantize":
        D = case["dim"]
        rows_of_scales = -(-B // BLOCK) if case["form"] == "weights" else B
        size = 4 if case["dtype"] == "fp32" else 2
        norm = 4 * D if case["form"] == "norm" else 0
        return {"bytes": B * D * (size + 1) + 4 * rows_of_scales * -(-D // BLOCK) + norm,
                "flops": B * D * (6 if case["form"] == "norm" else 2)}
    D, V, blocks = case["dim"], case["vocab"], -(-case["dim"] // BLOCK)
    scales = 4 * blocks * (B + -(-V // BLOCK))
    return {"bytes": (B + V) * D + scales + B * V * (4 if case["out"] == "fp32" else 2), "flops": 2 * B * D * V}


# ---- the definitions in 64 bits -------------------------------------------------------------

def _exact_sample(st):
    """By masks on normalised probabilities in vocabulary order, then a walk over them in falling order."""
    T, k, p, mp = _settings(st)
    z = st["logits"].double()
    z = torch.where(torch.isnan(z), -math.inf, z)
    B, V = z.shape
    order = torch.argsort(-z, dim=1, stable=True)
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=DEV).expand(B, V).contiguous())
    real = z > -math.inf
    greedy = ~(T >= GREEDY_BELOW)
    peak = z.amax(1, keepdim=True)
    rel = torch.where(z == peak, 0.0, (z - peak) / torch.where(greedy, 1.0, T))
    keep = real & torch.where(greedy, place < 1, True)
    keep &= torch.where((k > 0) & ~greedy, place < k, True)
    keep &= torch.where((mp > 0) & ~greedy, torch.exp(rel) >= mp.clamp(max=1.0), True)
    weight = torch.where(keep, torch.exp(rel), 0.0)
    prob = weight / weight.sum(1, keepdim=True)
    before = torch.cumsum(prob.gather(1, order), 1) - prob.gather(1, order)  # mass ahead of each place
    before = torch.empty_like(before).scatter_(1, order, before)
    keep &= torch.where((p > 0) & (p < 1) & ~greedy, before <= p, True)
    weight = torch.where(keep, weight, 0.0)
    prob = weight / weight.sum(1, keepdim=True)
    walk = torch.cumsum(prob.gather(1, order), 1)
    kept = keep.sum(1)
    coin = st["coins"].double().clamp(0.0, LARGEST_COIN)[:, None]
    at = torch.searchsorted(walk.nan_to_num(nan=1.0), coin, right=True).clamp(max=V - 1)
    at = torch.minimum(at, (kept[:, None] - 1).clamp(min=0))
    ids = order.gather(1, at)
    lp = torch.log(prob.gather(1, ids))
    none = (kept == 0)[:, None]
    return {"ids": torch.where(none, 0, ids)[:, 0].int(), "logprobs": torch.where(none, -math.inf, lp)[:, 0],
            "kept": kept.int()}


def _exact_quantize(st):
    x = st["x"].double()
    if st["case"]["form"] == "norm":
        w = st["norm_weight"].double()
        x = x / ((x ** 2).sum(1, keepdim=True) / x.shape[1] + EPS).sqrt() * w
    R, D = x.shape
    rows = torch.arange(R, device=DEV) // st["block_rows"]
    cols = torch.arange(D, device=DEV) // BLOCK
    peak = torch.zeros(int(rows[-1]) + 1, int(cols[-1]) + 1, dtype=torch.float64, device=DEV)
    by_col = torch.stack([c.abs().amax(1) for c in x.split(BLOCK, 1)], 1)
    peak.scatter_reduce_(0, rows[:, None].expand_as(by_col), by_col, "amax")
    scales = (peak / FP8_MAX).clamp(min=SMALLEST_SCALE)
    v = x / scales.float().double()[rows][:, cols]  # by the scale that is stored with the values
    # the nearest of the 8-bit values: 3 bits behind the leading one, steps of 2^-9 below 2^-6, ties to even
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(-6, 8)
    step = torch.exp2(e - 3)
    return {"values": (torch.round(v / step) * step).clamp(-FP8_MAX, FP8_MAX), "scales": scales}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(st)
    if case["kind"] == "quantize":
        return _exact_quantize(st)
    # the sum over the blocks of 128, each product scaled as it is added
    h, w = st["h"], st["w"]
    acc = torch.zeros(h.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    rows = torch.arange(w.shape[0], device=DEV) // BLOCK
    for b, at in enumerate(range(0, h.shape[1], BLOCK)):
        a = h[:, at:at + BLOCK].double() * st["h_scales"][:, b:b + 1].double()
        c = w[:, at:at + BLOCK].double() * st["w_scales"][rows, b:b + 1].double()
        acc += a @ c.t()
    return {"logits": acc}
