"""linear_lora around the change from the CUDA-core kernel to the tensor cores (one to five tokens),
against float64.

Tolerance: U and Y are rounded to the inputs' type once each (u = 2^-8 bf16, 2^-11 fp16: half a step is
u / 2 of the value; twice that is allowed) and sums of n fp32 products err by n 2^-24 of the sum of
magnitudes at most."""

import pytest
import torch

from latent_attn import functional

pytestmark = pytest.mark.gpu


def _check(got, x, W, A, B, ids, scales):
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -11
    x, W, A, B = (t.cpu().double() for t in (x, W, A, B))
    y, mag = x @ W.T, x.abs() @ W.abs().T
    slack = mag * x.shape[1] * 2.0 ** -24
    for m, a in enumerate(ids.tolist()):
        if 0 <= a < A.shape[0]:
            s = 1.0 if scales is None else float(scales[a])
            h = s * (A[a] @ x[m])
            y[m] += B[a] @ h
            hm = abs(s) * (A[a].abs() @ x[m].abs()) * (x.shape[1] + 2) * 2.0 ** -24 + h.abs() * u
            slack[m] += B[a].abs() @ hm + (B[a].abs() @ h.abs()) * B.shape[2] * 2.0 ** -24
    bound = slack + (y.abs() + slack) * u + 1e-30
    assert ((got.cpu().double() - y).abs() <= bound).all()


def _case(M, N, K, r, na, dtype, seed):
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()

    x, W = rnd(M, K), rnd(N, K, scale=K ** -0.5)
    A, B = rnd(na, r, K, scale=K ** -0.5), rnd(na, N, r, scale=r ** -0.5)
    ids = torch.randint(-1, na, (M,), generator=g, dtype=torch.int32).cuda()
    return x, W, A, B, ids


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K,r", [(1, 8, 8), (2, 264, 24), (77, 1000, 256), (513, 2056, 16), (9001, 264, 72),
                                   (1000, 16384, 40)])
def test_tokens(M, N, K, r, dtype):
    x, W, A, B, ids = _case(M, N, K, r, 3, dtype, M + N + K + r)
    scales = torch.tensor([0.5, -2.0, 1.0], device="cuda")
    _check(functional.linear_lora(x, W, A, B, ids, scales=scales), x, W, A, B, ids, scales)


@pytest.mark.parametrize("M", [1, 2])
def test_strided_tokens_and_broken_neighbours(M):
    """Rows of x with gaps, and infinities in the weights of adapters and tokens that are not the row's own."""
    x, W, A, B, _ = _case(M, 300, 520, 16, 4, torch.bfloat16, 5)
    wide = torch.full((M, 600), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :520] = x
    ids = torch.tensor([2, 0][:M], dtype=torch.int32, device="cuda")
    A[3], B[3], A[1], B[1] = float("inf"), float("nan"), float("nan"), float("inf")
    clean_a, clean_b = A.clone(), B.clone()
    clean_a[[1, 3]], clean_b[[1, 3]] = 0, 0
    got = functional.linear_lora(wide[:, :520], W, A, B, ids)
    _check(got, x, W, clean_a, clean_b, ids, None)
    if M == 2:
        ids[1] = 3
        got = functional.linear_lora(wide[:, :520], W, A, B, ids)
        assert not got[1].isfinite().any()
        _check(got[:1], x[:1], W, clean_a, clean_b, ids[:1], None)


def test_no_adapter_anywhere():
    x, W, A, B, _ = _case(2, 333, 1032, 8, 2, torch.float16, 6)
    ids = torch.tensor([-1, 7], dtype=torch.int32, device="cuda")
    _check(functional.linear_lora(x, W, A, B, ids), x, W, A, B, ids, None)
