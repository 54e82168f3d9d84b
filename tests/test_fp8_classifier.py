"""The 8-bit classifier: quantize_fp8 and rmsnorm_fp8 against their definition,
classifier_logits_fp8 against the product in 64 bits, and the decode step made
of them with sample_filtered.

Tolerances:
  * quantize_fp8: none.  The scale is one fp32 division, the value the nearest
    e4m3 of an fp32 division (torch does both on the CPU).
  * rmsnorm_fp8: fp32 arithmetic in front of the rounding.  A sum of D squares
    as a tree (a thread's run of at most 64, 8 levels), a mean, a square root,
    a reciprocal and two products: less than 2^-17 relative.  The scale is off
    by that and one division; a value by half a step of e4m3 (2^-4 relative, or
    2^-10 where the steps are 2^-9) plus that.
  * classifier_logits_fp8: products of e4m3 values are exact in fp32.  132
    additions at most make the sum of a block (128 products, 4 instructions),
    dim / 128 fold the blocks, each off by at most one fp32 step (2^-23) of the
    running sum, which the sum of the magnitudes bounds; as independent errors,
    the 2-norm of the result is off by the root of their number.  Plus half a
    step of the output's type.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

F8 = torch.float8_e4m3fn
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALLEST = 2.0 ** -126


def spread(s, R, D, block_rows):
    return s.repeat_interleave(block_rows, 0)[:R].repeat_interleave(128, 1)[:, :D]


def quantize_reference(x, block_rows):
    """Scales and values (as float32) on the CPU, from float32 x."""
    R, D = x.shape
    pad = torch.nn.functional.pad(x.abs(), (0, -D % 128, 0, -R % block_rows))
    blocks = pad.reshape(pad.shape[0] // block_rows, block_rows, pad.shape[1] // 128, 128)
    amax = blocks.amax(dim=(1, 3))
    s = (amax / 448.0).clamp(min=SMALLEST)
    s = torch.where(torch.isfinite(amax), s, torch.nan)
    q = (x / spread(s, R, D, block_rows)).clamp(-448.0, 448.0).to(F8)
    return q.float(), s


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("R,D", [(1, 1), (1, 128), (1, 4096), (3, 129), (5, 7), (127, 384), (128, 128), (129, 200),
                                 (300, 1000), (257, 4099), (2, 70000)])
def test_quantize(pkg, dtype, block_rows, R, D):
    g = torch.Generator().manual_seed(R * 7 + D)
    x = (torch.randn(R, D, generator=g) * torch.exp(2.0 * torch.randn(R, 1, generator=g))).to(dtype)
    q, s = pkg.quantize_fp8(x.cuda(), block_rows)
    torch.cuda.synchronize()
    want_q, want_s = quantize_reference(x.float(), block_rows)
    assert q.dtype == F8 and torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().float(), want_q)


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_values(pkg, block_rows, dtype):
    """Blocks of zeros, of the smallest and the largest numbers, with NaN and infinities (which show in their own
    block and nowhere else), and every tie between two e4m3 values."""
    R, D = 256, 1024
    x = torch.randn(R, D, generator=torch.Generator().manual_seed(1))
    x[0, :128] = 0.0
    x[128:, 128:256] = 0.0
    big, tiny = float(torch.finfo(dtype).max), float(torch.finfo(dtype).smallest_normal)
    x[:, 256:384] *= tiny * 64
    x[:, 384:512] = x[:, 384:512].sign() * big
    x[3, 520] = float("nan")
    x[130, 650] = float("inf")
    x[131, 651] = -float("inf")
    grid = torch.arange(0, 127, dtype=torch.uint8).view(F8).float()
    mids = (grid[:-1] + grid[1:]) / 2
    x[:, 768:896] = 448.0 * torch.ones(R, 128)
    x[:, 768:768 + 126] = mids
    x[7, 900:1000] = -0.0
    x = x.to(dtype)
    q, s = pkg.quantize_fp8(x.cuda(), block_rows)
    torch.cuda.synchronize()
    want_q, want_s = quantize_reference(x.float(), block_rows)
    assert same(s.cpu(), want_s) and same(q.cpu().float(), want_q)
    assert bool(torch.isnan(q[130, 640:768].float()).all()) and not bool(torch.isnan(q[2].float()).any()) == (block_rows == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D,ld,offset", [(5, 300, 301, 1), (130, 256, 264, 0), (130, 256, 257, 3), (4, 4096, 8192, 2)])
def test_quantize_strides_and_alignment(pkg, dtype, R, D, ld, offset):
    buf = torch.full((offset + R * ld,), float("nan"), dtype=dtype, device="cuda")
    x = buf[offset:].as_strided((R, D), (ld, 1))
    x.copy_(torch.randn(R, D, generator=torch.Generator().manual_seed(D)))
    for block_rows in (1, 128):
        shape = (-(-R // block_rows), -(-D // 128))
        qb = torch.zeros(R * D + 64 + offset, dtype=torch.uint8, device="cuda")
        sb = torch.full((shape[0] * shape[1] + 8,), -1.0, device="cuda")
        q, s = pkg.quantize_fp8(x, block_rows, out=qb[offset:offset + R * D].view(F8).view(R, D),
                                scales_out=sb[:shape[0] * shape[1]].view(shape))
        torch.cuda.synchronize()
        want_q, want_s = quantize_reference(x.float().cpu(), block_rows)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().float(), want_q)
        assert int(qb[offset + R * D:].sum()) == 0 and int(qb[:offset].sum()) == 0
        assert bool((sb[shape[0] * shape[1]:] == -1.0).all())
    w = 1.0 + 0.1 * torch.randn(D + 1, device="cuda")[1:]
    check_norm(pkg, x, w)


def check_norm(pkg, x, w):
    q, s = pkg.rmsnorm_fp8(x, w)
    torch.cuda.synchronize()
    R, D = x.shape
    xd = x.double()
    v = w.double() * xd / torch.sqrt((xd * xd).mean(1, keepdim=True) + 1e-5)
    pad = torch.nn.functional.pad(v.abs(), (0, -D % 128)).reshape(R, -1, 128)
    want_s = (pad.amax(2) / 448.0).clamp(min=SMALLEST)
    slop = 2.0 ** -17
    assert bool(((s.double() - want_s).abs() <= slop * want_s).all())
    t = v / spread(s.double(), R, D, 1)
    err = (q.double() - t).abs()
    assert bool((err <= torch.clamp(t.abs() * 2.0 ** -4, min=2.0 ** -10) + slop * t.abs()).all()), float(err.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D", [(1, 1), (1, 128), (1, 4096), (3, 130), (7, 4100), (33, 1104), (2, 8192), (2, 8200),
                                 (2, 16384), (2, 20001)])
def test_rmsnorm(pkg, dtype, B, D):
    g = torch.Generator().manual_seed(B + D)
    x = (3.0 * torch.randn(B, D, generator=g)).to(dtype).cuda()
    check_norm(pkg, x, (1.0 + 0.1 * torch.randn(D, generator=g)).cuda())
    if B > 1:
        x[1] = 0.0
        check_norm(pkg, x, torch.ones(D, device="cuda"))


@pytest.mark.gpu
def test_rmsnorm_poisons_its_own_row_only(pkg):
    x = torch.randn(4, 512, device="cuda")
    x[1, 77] = float("nan")
    q, s = pkg.rmsnorm_fp8(x, torch.ones(512, device="cuda"))
    torch.cuda.synchronize()
    bad = torch.isnan(s).any(1).tolist()
    assert bad == [False, True, False, False] and bool(torch.isnan(q[1].float()).all())


def operands(B, D, V, seed):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(B, D, generator=g) * torch.exp(torch.randn(B, 1, generator=g))
    w = torch.randn(V, D, generator=g) * 0.02 * torch.exp(torch.randn(V, 1, generator=g))
    hq, hs = quantize_reference(h, 1)
    wq, ws = quantize_reference(w, 128)
    # every block its own scale, not only its own row's: what a wrong block's scale would give shows
    hs = hs * torch.exp2(torch.randint(-2, 3, hs.shape, generator=g).float())
    ws = ws * torch.exp2(torch.randint(-2, 3, ws.shape, generator=g).float())
    return hq.to(F8).cuda(), hs.cuda(), wq.to(F8).cuda(), ws.cuda()


def check_logits(h, hs, w, ws, got):
    B, D = h.shape
    V = w.shape[0]
    a = h.double() * spread(hs.double(), B, D, 1)
    c = w.double() * spread(ws.double(), V, D, 128)
    ref, mag = a @ c.t(), a.abs() @ c.abs().t()
    n = 132 + -(-D // 128)
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    err = (got.double() - ref).abs()
    assert bool((err <= n * 2.0 ** -23 * mag + half * ref.abs() + 1e-30).all()), float((err / mag).max())
    rel = float(err.norm() / ref.norm())
    assert rel <= math.sqrt(n) * 2.0 ** -22 + (half if half > 1e-4 else 2.0 ** -24), rel


SHAPES = [(1, 4096, 32000), (2, 128, 1), (1, 16, 5), (3, 144, 257), (8, 1104, 4099), (16, 512, 130), (17, 4096, 999),
          (32, 2048, 2050), (33, 640, 300), (64, 272, 1000), (65, 512, 700), (100, 1040, 520), (128, 384, 256),
          (129, 400, 257), (200, 4096, 1024), (300, 1104, 2051), (517, 256, 771), (1, 16384, 640), (70, 16400, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,V", SHAPES)
def test_logits(pkg, B, D, V, out):
    ops = operands(B, D, V, B + D + V)
    pad = 3 if V % 2 else 8
    buf = torch.full((B + 1, V + pad), -5.0, dtype=out, device="cuda")
    got = pkg.classifier_logits_fp8(*ops, logits_out=buf[:B, :V])
    torch.cuda.synchronize()
    check_logits(*ops, got)
    assert bool((buf[B] == -5.0).all()) and bool((buf[:, V:] == -5.0).all())
    dense = pkg.classifier_logits_fp8(*ops, logits_out=torch.empty(B, V, dtype=out, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(dense, got)


@pytest.mark.gpu
def test_logits_of_the_whole_range_of_values(pkg):
    """Every e4m3 value meets every other, zeros and the signs of zero among them."""
    all_q = torch.arange(256, dtype=torch.uint8)
    finite = all_q[(all_q & 0x7F) != 0x7F]
    g = torch.Generator().manual_seed(2)
    h = finite[torch.randint(0, len(finite), (40, 384), generator=g)].view(F8).cuda()
    w = finite[torch.randint(0, len(finite), (300, 384), generator=g)].view(F8).cuda()
    hs, ws = torch.ones(40, 3, device="cuda"), torch.ones(3, 3, device="cuda")
    got = pkg.classifier_logits_fp8(h, hs, w, ws)
    torch.cuda.synchronize()
    check_logits(h, hs, w, ws, got)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [4, 40, 200])
def test_a_nan_row_stays_in_its_row(pkg, B):
    h, hs, w, ws = operands(B, 512, 400, 3)
    hs[2, 1] = float("nan")
    got = pkg.classifier_logits_fp8(h, hs, w, ws)
    torch.cuda.synchronize()
    bad = torch.isnan(got)
    assert bool(bad[2].all()) and int(bad.sum()) == 400


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 20, 150])
def test_logits_repeat_and_graph(pkg, B):
    ops = operands(B, 1024, 3001, 9)
    want = pkg.classifier_logits_fp8(*ops).clone()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.classifier_logits_fp8(*ops, logits_out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,norm,logits", [(1, True, None), (5, False, torch.bfloat16), (40, True, torch.float32),
                                           (200, True, torch.bfloat16), (130, False, None)])
def test_decode_step_is_its_parts(pkg, dtype, B, norm, logits):
    D, V = 1024, 3001
    g = torch.Generator().manual_seed(B)
    x = (2.0 * torch.randn(B, D, generator=g)).to(dtype).cuda()
    nw = (1.0 + 0.1 * torch.randn(D, generator=g)).cuda() if norm else None
    wq, ws = pkg.quantize_fp8((torch.randn(V, D, generator=g) * 0.05).cuda(), 128)
    coins = torch.rand(B, generator=g).cuda()
    lg = None if logits is None else torch.empty(B, V, dtype=logits, device="cuda")
    lp, kept = torch.empty(B, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    ids = pkg.classifier_fp8_sample_filtered(x, nw, wq, ws, 0.8, 50, 0.95, 0.01, coins=coins, logits_out=lg,
                                             logprobs_out=lp, kept_out=kept)
    q, s = pkg.rmsnorm_fp8(x, nw) if norm else pkg.quantize_fp8(x)
    want_lg = pkg.classifier_logits_fp8(q, s, wq, ws, logits_out=None if lg is None else torch.empty_like(lg))
    lp2, kept2 = torch.empty_like(lp), torch.empty_like(kept)
    want = pkg.sample_filtered(want_lg, 0.8, 50, 0.95, 0.01, coins=coins, logprobs_out=lp2, kept_out=kept2)
    torch.cuda.synchronize()
    assert torch.equal(ids, want) and torch.equal(lp, lp2) and torch.equal(kept, kept2)
    if lg is not None:
        assert torch.equal(lg, want_lg)


@pytest.mark.gpu
def test_decode_loop_in_a_graph(pkg):
    """Steps whose next input is gathered on the device from the sampled ids: eager, and captured once and
    replayed.  A second graph with a workspace of its own runs between the replays."""
    B, D, V, steps = 24, 256, 2048, 5
    g = torch.Generator().manual_seed(41)
    table = (torch.randn(V, D, generator=g) * 2.0).cuda()
    nw = (1.0 + 0.1 * torch.randn(D, generator=g)).cuda()
    wq, ws = pkg.quantize_fp8(table, 128)
    seeds = torch.from_numpy(pkg.workloads.row_seeds(B).view(np.int64).copy()).cuda()
    ids0 = torch.arange(B, dtype=torch.int32, device="cuda") * 37 % V

    def step(x, st, ids):
        pkg.classifier_fp8_sample_filtered(x, nw, wq, ws, 0.9, 0, 0.9, 0.0, st, out_ids=ids)
        pkg.gather_rows(table, ids, out=x)

    def run(fn, x, st, ids):
        out = []
        for _ in range(steps):
            fn(x, st, ids)
            out.append(ids.clone())
        torch.cuda.synchronize()
        return torch.stack(out).cpu(), st.cpu()

    want = run(step, pkg.gather_rows(table, ids0), seeds.clone(), torch.empty(B, dtype=torch.int32, device="cuda"))
    graphs = []
    for _ in range(2):
        x, st = pkg.gather_rows(table, ids0), seeds.clone()
        ids = torch.empty(B, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(x, st, ids)
        x.copy_(pkg.gather_rows(table, ids0))
        st.copy_(seeds)
        graphs.append((graph, x, st, ids))
    torch.cuda.synchronize()

    def both(x, st, ids):
        graphs[0][0].replay()
        graphs[1][0].replay()

    got = run(both, *graphs[0][1:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(graphs[1][3].cpu(), want[0][-1])
    assert len(set(want[0][-1].tolist())) > 1


@pytest.mark.gpu
def test_side_stream_without_library_buffers(pkg):
    """The decode step on a stream that is not the current one, while torch's allocator is busy with others."""
    B, D, V = 16, 512, 4000
    x = torch.randn(B, D, device="cuda")
    wq, ws = pkg.quantize_fp8(torch.randn(V, D, device="cuda") * 0.05, 128)
    coins = torch.rand(B, device="cuda")
    want = pkg.classifier_fp8_sample_filtered(x, None, wq, ws, 0.9, 0, 0.9, 0.0, coins=coins).clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    outs = []
    for _ in range(30):
        outs.append(pkg.classifier_fp8_sample_filtered(x, None, wq, ws, 0.9, 0, 0.9, 0.0, coins=coins, stream=s))
        torch.full((B * D + 4096,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


@pytest.mark.gpu
def test_python_refusals(pkg):
    h, hs, w, ws = operands(4, 128, 300, 1)
    x = torch.zeros(4, 128, device="cuda")
    out = torch.empty(4, 300, dtype=torch.float16, device="cuda")
    c = torch.zeros(4, device="cuda")
    bad = [
        lambda: pkg.quantize_fp8(x.double()),
        lambda: pkg.quantize_fp8(x.cpu()),
        lambda: pkg.quantize_fp8(x, 64),
        lambda: pkg.quantize_fp8(x.t()),
        lambda: pkg.quantize_fp8(x, out=torch.empty(4, 127, dtype=F8, device="cuda")),
        lambda: pkg.quantize_fp8(x, scales_out=torch.empty(4, 2, device="cuda")),
        lambda: pkg.rmsnorm_fp8(x, c),
        lambda: pkg.classifier_logits_fp8(h.float(), hs, w, ws),
        lambda: pkg.classifier_logits_fp8(h, hs, w.view(torch.uint8), ws),
        lambda: pkg.classifier_logits_fp8(h, hs[:3], w, ws),
        lambda: pkg.classifier_logits_fp8(h, hs, w, ws[:2]),
        lambda: pkg.classifier_logits_fp8(h, hs, w[:, :64].contiguous(), ws),
        lambda: pkg.classifier_logits_fp8(h, hs, w, ws, logits_out=out),
        lambda: pkg.classifier_logits_fp8(h, hs, w, ws, logits_out=out.float()[:3]),
        lambda: pkg.classifier_logits_fp8(*operands(2, 120, 64, 1)),
        lambda: pkg.classifier_fp8_sample_filtered(x.t(), None, w, ws, 1.0, 0, 1.0, 0.0, coins=c),
        lambda: pkg.classifier_fp8_sample_filtered(x, None, w, ws, 1.0, 0, 1.0, 0.0),
        lambda: pkg.classifier_fp8_sample_filtered(x, None, w, ws, 1.0, 0, 1.0, 0.0, coins=c, logits_out=out),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(pkg.SamplerError):
            f()
            pytest.fail(f"call {i} was not refused")
    assert pkg.quantize_fp8(x[:0])[0].shape == (0, 128)
    assert pkg.classifier_logits_fp8(h[:0], hs[:0], w, ws).shape == (0, 300)


def test_c_refusals_before_any_device_work(pkg):
    """Arguments are checked before a device is touched (the addresses passed are never read)."""
    L = pkg.lib()
    A = 4096

    def quant(x=A, dt=0, rows=2, dim=256, ld=256, block=1, q=A, s=A):
        return L.quantize_fp8(x, dt, rows, dim, ld, block, q, s, None)

    assert [quant(x=None), quant(q=None), quant(s=None), quant(dt=3), quant(rows=-1), quant(dim=0), quant(ld=255),
            quant(block=64), quant(x=A + 2), quant(dt=1, x=A + 1), quant(s=A + 2)] == [-1] * 11
    assert quant(dim=(1 << 24) + 1, ld=1 << 30) == -2
    assert quant(rows=0) == 0
    assert L.rmsnorm_fp8(A, 0, None, 2, 256, 256, A, A, None) == -1
    assert L.rmsnorm_fp8(A, 0, A + 1, 2, 256, 256, A, A, None) == -1

    def gemm(h=A, hs=A, w=A, ws=A, b=2, d=256, v=100, out=A, dt=0, ld=100):
        return L.classifier_logits_fp8(h, hs, w, ws, b, d, v, out, dt, ld, None)

    assert [gemm(h=None), gemm(hs=None), gemm(w=None), gemm(ws=None), gemm(out=None), gemm(b=-1), gemm(d=8),
            gemm(d=100), gemm(v=0), gemm(ld=99), gemm(dt=2), gemm(h=A + 8), gemm(w=A + 8), gemm(hs=A + 2),
            gemm(out=A + 2)] == [-1] * 15
    assert gemm(d=1 << 17) == -2 and gemm(v=(1 << 30) + 1, ld=1 << 31) == -2
    assert gemm(b=0) == 0

    cfg = pkg.SamplerFilterConfig(100, 0, 1.0, 0, 1.0, 0.0)
    need = L.classifier_fp8_workspace_bytes(2, 256, 100, 0)
    assert need == 512 + 256 + 2 * 100 * 4 and L.classifier_fp8_workspace_bytes(2, 256, 100, -1) == 768
    assert L.classifier_fp8_workspace_bytes(0, 256, 100, 0) == 0

    def step(c=cfg, x=A, dt=0, w=A, ws=A, b=2, d=256, coins=A, ids=A, wsp=A, n=need, out=None):
        return L.classifier_fp8_sample_filtered(None if c is None else ctypes.byref(c), x, dt, None, w, ws, b, d, None,
                                                None, None, None, coins, None, ids, None, None, out, None, wsp, n, None)

    f16 = pkg.SamplerFilterConfig(100, 2, 1.0, 0, 1.0, 0.0)
    assert [step(c=None), step(x=None), step(w=None), step(ws=None), step(coins=None), step(ids=None), step(dt=5),
            step(d=100), step(c=f16), step(w=A + 8), step(out=A + 1), step(wsp=A + 8)] == [-1] * 12
    assert step(n=need - 1) == -4 and step(wsp=None) == -4
    assert step(d=1 << 17) == -2
    assert step(b=0) == 0
