"""Attention of few rows over many keys: the joins of the keys' parts, on both sides of the sizes at which a
row takes a block, against the formula in 64 bits (tolerances as in test_gpu_attention)."""
import pytest
import torch

from test_gpu_attention import DTYPES, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,Nq,Nk,D,live", [
    (1, 1, 1, 1, 8040, 4, 1.0), (1, 2, 1, 1, 5001, 16, 0.9), (2, 2, 2, 1, 2100, 33, 1.0),
    (1, 8, 2, 1, 8040, 128, 0.5), (8, 4, 1, 8, 1030, 64, 0.9), (1, 1, 1, 257, 4100, 64, 1.0),
    (1, 4, 4, 1, 6000, 96, 0.003), (3, 1, 1, 2, 4099, 1, 0.9), (1, 16, 16, 16, 1200, 32, 1.0)])
def test_few_rows(B, Hq, Hkv, Nq, Nk, D, live, dtype):
    print(f"[attend] join B={B} H={Hq}/{Hkv} {Nq}x{Nk} D={D} {dtype}", flush=True)
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, dtype)
    mask = None
    if live < 1:
        gen = torch.Generator(device="cuda").manual_seed(5)
        mask = torch.rand(B, Nk, device="cuda", generator=gen) < live
        mask[B - 1, : Nk // 2] = False          # parts without a key
        mask[B - 1, -1] = True
    check(q, k, v, do, mask)
