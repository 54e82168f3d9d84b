"""A device wait of the 8-bit decode step that runs out: the rows it leaves without
logits are reported, not sampled from what the buffer held, and the device stays
usable.  The wait is made to run out by a self-test form of the product that issues
none (nothing is left in flight); no GPU fault is involved.
"""
import ctypes

import numpy as np
import pytest
import torch

SAMPLER_E_DEVICE = -6


def test_selftest_refusals(pkg):
    L = pkg.lib()
    flag = ctypes.c_int(0)
    assert L.classifier_fp8_selftest_wait_timeout(0, ctypes.byref(flag)) == -1
    assert L.classifier_fp8_selftest_wait_timeout((1 << 24) + 1, ctypes.byref(flag)) == -1
    assert L.classifier_fp8_selftest_wait_timeout(16, None) == -1


@pytest.mark.gpu
def test_a_timeout_of_the_product_flags_its_rows(pkg):
    L = pkg.lib()
    flag = ctypes.c_int(-1)
    rc = L.classifier_fp8_selftest_wait_timeout(1 << 10, ctypes.byref(flag))
    assert rc == SAMPLER_E_DEVICE, L.sampler_last_error()
    assert flag.value == pkg.ROW_TIMEOUT
    assert b"bounded device wait" in L.sampler_last_error()
    s = pkg.build_sampler(32000, 0.7, 0.9, 42)  # a synchronous call sees no stale error
    assert pkg.sample(s, np.zeros(32000, np.float32)) >= 0
    pkg.free_sampler(s)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("B", [1, 7, 130])
def test_what_the_outputs_held_before_does_not_matter(pkg, B, norm):
    """out_ids, and the logits of an earlier step, may hold anything before the call."""
    g = torch.Generator().manual_seed(B)
    D, V = 272, 999
    x = torch.randn(B, D, generator=g).cuda()
    nw = torch.ones(D, device="cuda") if norm else None
    wq, ws = pkg.quantize_fp8((torch.randn(V, D, generator=g) * 0.05).cuda(), 128)
    coins = torch.rand(B, generator=g).cuda()
    got = []
    for before in (-1, 5, -(1 << 31)):
        ids = torch.full((B + 2,), before, dtype=torch.int32, device="cuda")
        flags = torch.full((B,), -7, dtype=torch.int32, device="cuda")
        pkg.classifier_fp8_sample_filtered(x, nw, wq, ws, 0.8, 0, 0.9, 0.0, coins=coins, out_ids=ids[:B], row_flags=flags)
        torch.cuda.synchronize()
        assert flags.tolist() == [0] * B and ids[B:].tolist() == [before] * 2
        got.append(ids[:B].tolist())
    assert got[0] == got[1] == got[2]
