"""The 8-bit decode step with every setting by row and every output asked for,
against its parts."""
import numpy as np
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("logits", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [1, 33, 300, 700])
def test_settings_and_outputs_by_row(pkg, B, logits):
    D, V = 528, 5003
    g = torch.Generator().manual_seed(B)
    rng = np.random.default_rng(B)
    x = (2.0 * torch.randn(B, D, generator=g)).cuda()
    if B > 4:
        x[3, 7] = float("nan")    # a row whose logits are all NaN
        x[4, 8] = float("inf")
    nw = (1.0 + 0.1 * torch.randn(D, generator=g)).cuda()
    wq, ws = pkg.quantize_fp8((torch.randn(V, D, generator=g) * 0.1).cuda(), 128)
    col = lambda v, dt: torch.from_numpy(rng.choice(v, B).astype(dt)).cuda()  # noqa: E731
    rows = dict(temperature_rows=col([0.0, 0.3, 0.8, 1.0, 2.0, -1.0], np.float32), topk_rows=col([0, 1, 5, 50, 2 * V, -3], np.int32),
                topp_rows=col([0.0, 0.5, 0.9, 1.0, 2.0], np.float32), minp_rows=col([0.0, 0.01, 0.3, 1.0], np.float32))
    seeds = torch.from_numpy(pkg.workloads.row_seeds(B).view(np.int64).copy()).cuda()

    def outputs():
        return dict(logprobs_out=torch.full((B,), 9.0, device="cuda"), kept_out=torch.full((B,), -9, dtype=torch.int32, device="cuda"),
                    row_flags=torch.full((B,), -9, dtype=torch.int32, device="cuda"),
                    out_ids=torch.full((B,), -9, dtype=torch.int32, device="cuda"))

    lg, st, got = torch.empty(B, V, dtype=logits, device="cuda"), seeds.clone(), outputs()
    pkg.classifier_fp8_sample_filtered(x, nw, wq, ws, 0.5, 3, 0.5, 0.5, st, logits_out=lg, **rows, **got)
    want_lg, want_st, want = torch.empty_like(lg), seeds.clone(), outputs()
    pkg.classifier_logits_fp8(*pkg.rmsnorm_fp8(x, nw), wq, ws, logits_out=want_lg)
    pkg.sample_filtered(want_lg, 0.5, 3, 0.5, 0.5, want_st, **rows, **want)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(lg.float()), torch.nan_to_num(want_lg.float())) and torch.equal(st, want_st)
    for name in got:
        assert torch.equal(got[name], want[name]), name
    flags = got["row_flags"].tolist()
    bad = pkg.ROW_NAN | pkg.ROW_NO_CANDIDATE
    assert flags == [bad if B > 4 and b in (3, 4) else 0 for b in range(B)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_a_row_whose_squares_overflow(pkg, dtype):
    """fp32 squares, as in rmsnorm_bf16: 1 / sqrt(infinity) makes the row zeros, and no other row."""
    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    x[1] *= 1e20
    q, s = pkg.rmsnorm_fp8(x, torch.ones(700, device="cuda"))
    torch.cuda.synchronize()
    assert not bool(q[1].float().any()) and bool((s[1] == 2.0 ** -126).all())
    assert bool((q[[0, 2]].float().abs().amax(1) == 448.0).all())
