"""The 8-bit classifier where offsets pass 32 bits: rows of a strided or large
input, values, weights and logits that start beyond 2^31 elements.  The last rows are
compared with a small call on the same rows, which other tests hold to the definition.
"""
import pytest
import torch

from test_fp8_classifier import F8, operands, quantize_reference, spread

PAST = 2 ** 31


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_inputs(pkg, dtype):
    R, D, ld = 5, 300, 600_000_000
    buf = torch.empty((R - 1) * ld + D, dtype=dtype, device="cuda")
    x = buf.as_strided((R, D), (ld, 1))
    rows = torch.randn(R, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    x.copy_(rows)
    w = torch.ones(D, device="cuda")
    for block_rows in (1, 128):
        q, s = pkg.quantize_fp8(x, block_rows)
        want_q, want_s = quantize_reference(rows.float(), block_rows)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().float(), want_q)
    a, b = pkg.rmsnorm_fp8(x, w), pkg.rmsnorm_fp8(rows.cuda(), w)
    torch.cuda.synchronize()
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["rows", "weights", "norm"])
def test_values_past_two_to_the_31(pkg, form):
    R, D = 32900, 65537 if form == "weights" else 65544  # ragged and whole rows
    assert (R - 200) * D < PAST < (R - 100) * D
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(260, D, generator=g, device="cuda").bfloat16()
    x[-260:] = tail
    w = torch.ones(D, device="cuda")
    call = {"rows": lambda t: pkg.quantize_fp8(t), "weights": lambda t: pkg.quantize_fp8(t, 128),
            "norm": lambda t: pkg.rmsnorm_fp8(t, w)}[form]
    q, s = call(x)
    first = R // 128 * 128 - 128  # a block row of the weights' form
    want_q, want_s = call(x[first:].clone())
    torch.cuda.synchronize()
    assert torch.equal(q[first:].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[-want_s.shape[0]:], want_s)
    assert not bool(q[:1000].view(torch.uint8).any())


@pytest.mark.gpu
@pytest.mark.parametrize("out,ld", [(torch.float32, 600_000_000), (torch.bfloat16, 600_000_001)])
def test_strided_logits(pkg, out, ld):
    B, D, V = 5, 256, 700
    ops = operands(B, D, V, 4)
    buf = torch.empty((B - 1) * ld + V + 8, dtype=out, device="cuda")
    got = buf.as_strided((B, V), (ld, 1))
    ends = [buf[b * ld + V: b * ld + V + 8] for b in range(B)]
    for e in ends:
        e.fill_(-5.0)
    want = pkg.classifier_logits_fp8(*ops, logits_out=torch.empty(B, V, dtype=out, device="cuda"))
    pkg.classifier_logits_fp8(*ops, logits_out=got)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(bool((e == -5.0).all()) for e in ends)


@pytest.mark.gpu
def test_weights_past_two_to_the_31(pkg):
    B, D, V = 3, 16384, 131400
    assert (V - 500) * D < PAST < V * D
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.zeros(V, D, dtype=torch.uint8, device="cuda")
    w[-640:] = torch.randint(0, 120, (640, D), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.ones((V + 127) // 128, D // 128, device="cuda")
    ws[-5:] = torch.rand(5, D // 128, generator=g, device="cuda")
    h, hs = pkg.quantize_fp8(torch.randn(B, D, generator=g, device="cuda"))
    got = pkg.classifier_logits_fp8(h, hs, w.view(F8), ws)
    first = V // 128 * 128 - 512
    want = pkg.classifier_logits_fp8(h, hs, w[first:].clone().view(F8), ws[first // 128:].clone())
    torch.cuda.synchronize()
    assert torch.equal(got[:, first:], want)
    a = h.double() * spread(hs.double(), B, D, 1)
    c = w[-100:].view(F8).double() * spread(ws.double()[first // 128:], V - first, D, 128)[-100:]
    ref, mag = a @ c.t(), a.abs() @ c.abs().t()  # 132 additions a block and a fold of 128 blocks, a step each
    assert bool(((got[:, -100:].double() - ref).abs() <= (132 + D // 128) * 2.0 ** -23 * mag).all())
    assert not bool(got[:, :1000].any())


@pytest.mark.gpu
def test_decode_step_with_logits_past_two_to_the_31(pkg):
    B, D, V = 70000, 128, 32000
    assert (B - 4000) * V < PAST < (B - 2000) * V
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(B, D, generator=g, device="cuda").bfloat16()
    wq, ws = pkg.quantize_fp8(torch.randn(V, D, generator=g, device="cuda") * 0.2, 128)
    coins = torch.rand(B, generator=g, device="cuda")
    flags = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    logits = torch.empty(B, V, dtype=torch.bfloat16, device="cuda")
    ids = pkg.classifier_fp8_sample_filtered(x, None, wq, ws, 0.9, 40, 0.9, 0.0, coins=coins, logits_out=logits, row_flags=flags)
    few = slice(B - 1024, B)
    want_logits = torch.empty(1024, V, dtype=torch.bfloat16, device="cuda")
    want = pkg.classifier_fp8_sample_filtered(x[few].clone(), None, wq, ws, 0.9, 40, 0.9, 0.0, coins=coins[few].clone(),
                                              logits_out=want_logits)
    torch.cuda.synchronize()
    assert torch.equal(ids[few], want) and torch.equal(logits[few], want_logits) and not bool(flags.any())
