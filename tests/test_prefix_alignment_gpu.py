"""mla_prefix_decode with inputs at addresses that are multiples of 16 bytes but not of 32, and with many
groups of one tile: the same bits as with aligned inputs, and the float64 result.

Tolerance of the float64 comparison (bf16, |scores| < 8): P, records and result are rounded by 2^-9 of
their size at most, fp16 partial scores move a weight by 2^-11 * 8 * ln 2 * 2 < 2^-7.5 of itself in
either direction; all of them together stay below 2e-2 of the largest output."""

import math

import pytest
import torch

from latent_attn import MLAConfig, functional

pytestmark = pytest.mark.gpu

DC, DR = 512, 64


def _shifted(t):
    """The same values 16 bytes past an aligned address."""
    buf = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    buf[8:] = t.reshape(-1)
    view = buf[8:].view(t.shape)
    assert view.data_ptr() % 32 == 16
    return view


@pytest.mark.parametrize("heads", [5, 16, 64, 128])
def test_shifted_queries(heads):
    g = torch.Generator().manual_seed(heads)
    B, plen = 23, 130
    lens = [(7 * b) % 80 for b in range(B)]
    offs = [0] * B
    at = 200
    for b in range(B):
        offs[b] = at
        at += lens[b]
    dt = torch.bfloat16
    kv = torch.randn(at, DC + DR, generator=g).to(dt).cuda()
    qa = (torch.randn(B, heads, DC, generator=g) * 0.5).to(dt).cuda()
    qr = torch.randn(B, heads, DR, generator=g).to(dt).cuda()
    cfg = MLAConfig(512, DC, 128, DR, heads, 128)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    kw = dict(group_starts=i32([0, 11, B]), prefix_lens=i32([plen, 64]), max_prefix_len=plen, seq_lens=i32(lens),
              max_seq_len=80, prefix_offsets=torch.tensor([0, 40], device="cuda"),
              kv_offsets=torch.tensor(offs, device="cuda"))
    want = functional.mla_prefix_decode(kv, qa, qr, cfg, **kw)
    got = functional.mla_prefix_decode(_shifted(kv), _shifted(qa), _shifted(qr), cfg, **kw)
    assert torch.equal(got, want)
    k = kv.double().cpu()
    worst = top = 0.0
    for b in range(B):
        first, n = (0, plen) if b < 11 else (40, 64)
        rows = torch.cat([k[first:first + n], k[offs[b]:offs[b] + lens[b]]])
        s = torch.cat([qa[b], qr[b]], 1).double().cpu() @ rows.T / math.sqrt(128 + DR)
        o = torch.softmax(s, 1) @ rows[:, :DC]
        worst = max(worst, float((got[b].double().cpu() - o).abs().max()))
        top = max(top, float(o.abs().max()))
    assert worst <= 2e-2 * top
