"""mla_cache_append_rope against its definition in 64 bits: ragged batches of prompts and single
tokens, both cache layouts, the norm, tables and computed angles, strided inputs, the element path
of odd dimensions, and the cases that must write nothing.

Tolerance: an output is one rounding of an fp32 result, so it lies within half a unit in the last
place of the exact value plus the fp32 error. For bf16 (8 significant bits) that is at most 2^-8 of
the value, for fp16 2^-11, plus 2^-18 of the row's largest magnitude for the fp32 arithmetic and, with computed angles,
8e-7 of it for cos and sin (their documented bound is 6e-7)."""

import numpy as np
import pytest
import torch

from latent_attn import MLAConfig
from latent_attn.functional import mla_cache_append_rope
from latent_attn.synthetic import build_rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _exact(c, k, q, cu, lens, cap, rows, row_of, dims, cos, sin, w, eps, before):
    """(cache, q_out, new_lens) in float64; `row_of(b, p)` is the cache row of a position or None."""
    dc, dR, H = dims
    cache, qo = before.double().clone(), torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    new = []
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        new.append(lens[b] if lens[b] < 0 or lens[b] >= cap else min(cap, lens[b] + n))
        for i in range(n):
            t, p = cu[b] + i, lens[b] + i
            if lens[b] < 0 or p >= cap:
                continue
            co, si = cos[p], sin[p]

            def rot(x):
                a, bb = x[..., :dR // 2], x[..., dR // 2:]
                return torch.cat([a * co - bb * si, a * si + bb * co], -1)
            x = c[t].double()
            if w is not None:
                x = x / torch.sqrt((x * x).mean() + eps) * w.double()
            r = row_of(b, p)
            if r is not None and 0 <= r < rows:
                cache[r] = torch.cat([x, rot(k[t].double())])
            if q is not None:
                qo[t] = rot(q[t].double())
    return cache, qo, new


def _near(got, want, dtype, slack):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    top = want.abs().amax(-1, keepdim=True)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0       # half of fp16's smallest subnormal
    err = (got - want).abs() - half * want.abs() - (2.0 ** -18 + slack) * top - tiny
    assert float(err.max()) <= 0, float(err.max())


def _tables(n, dR, theta=10000.0):
    freq = torch.tensor([np.float32(theta ** (-2.0 * i / dR)) for i in range(dR // 2)], dtype=torch.float64)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * freq[None]
    return ang.cos(), ang.sin()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dims", [(512, 64, 16), (512, 64, 128), (96, 32, 5), (20, 6, 3), (1024, 96, 2)])
@pytest.mark.parametrize("paged,norm,tables", [(True, True, True), (False, False, False), (False, True, True),
                                               (True, False, False)])
def test_ragged_batch(dtype, dims, paged, norm, tables):
    dc, dR, H = dims
    g = torch.Generator().manual_seed(dc + dR + H)
    counts, lens = [0, 1, 70, 0, 3, 64, 1], [5, 0, 63, 0, 130, 64, 199]
    cap, page = 200, 24                                        # pages that end anywhere
    B, T = len(counts), sum(counts)
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    pages = -(-cap // page)
    table = torch.randperm(B * pages + 3, generator=g)[:B * pages].view(B, pages).to(torch.int32)
    rows = (B * pages + 3) * page if paged else B * cap + 7
    offs = torch.tensor([b * cap + 7 for b in range(B)], dtype=torch.int64)
    before = torch.randn(rows, dc + dR, generator=g).to(dtype)
    # c and k_rope as slices of one projection's output, the queries as a slice of wider heads
    proj = (3 * torch.randn(T, dc + dR + 8, generator=g)).to(dtype)
    heads = torch.randn(T, H, dR + 16, generator=g).to(dtype)
    w = (1 + 0.1 * torch.randn(dc, generator=g)).to(dtype) if norm else None
    cos, sin = build_rope_tables(cap, dR) if tables else _tables(cap, dR)
    kv, projd, headsd = before.to(DEV), proj.to(DEV), heads.to(DEV)
    new, status = torch.full((B,), -7, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cfg = MLAConfig(0, dc, 128, dR, H, 128)
    kw = dict(page_table=table.to(DEV), page_rows=page) if paged else dict(kv_offsets=offs.to(DEV))
    q = mla_cache_append_rope(kv, projd[:, :dc], projd[:, dc:dc + dR], torch.tensor(cu, dtype=torch.int32, device=DEV),
                              torch.tensor(lens, dtype=torch.int32, device=DEV), cap, cfg,
                              rope_cos=cos.float().to(DEV) if tables else None,
                              rope_sin=sin.float().to(DEV) if tables else None,
                              norm_weight=w.to(DEV) if norm else None, norm_eps=1e-5, q_rope=headsd[..., 8:8 + dR],
                              new_lens=new, status=status, **kw)

    def row_of(b, p):
        return int(table[b, p // page]) * page + p % page if paged else int(offs[b]) + p
    want, qw, nl = _exact(proj[:, :dc], proj[:, dc:dc + dR], heads[..., 8:8 + dR], cu, lens, cap, rows, row_of, dims,
                          cos.double(), sin.double(), w, 1e-5, before)
    slack = 0.0 if tables else 8e-7
    _near(kv[:, :dc], want[:, :dc], dtype, 0.0)
    _near(kv[:, dc:], want[:, dc:], dtype, slack)
    _near(q, qw, dtype, slack)
    assert new.tolist() == nl and int(status) == 0
    assert torch.equal(headsd.cpu(), heads)                    # the input is left alone


def test_in_place_queries_and_default_layout():
    g = torch.Generator().manual_seed(3)
    B, cap, H = 3, 40, 32
    cfg = MLAConfig(0, 512, 128, 64, H, 128)
    c, k = torch.randn(B, 512, generator=g).bfloat16().to(DEV), torch.randn(B, 64, generator=g).bfloat16().to(DEV)
    q = torch.randn(B, H, 64, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([0, 39, 7], dtype=torch.int32, device=DEV)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    kv = torch.zeros(B * cap, 576, dtype=torch.bfloat16, device=DEV)
    apart = mla_cache_append_rope(kv, c, k, cu, lens, cap, cfg, q_rope=q)
    again = kv.clone()
    got = mla_cache_append_rope(kv, c, k, cu, lens, cap, cfg, q_rope=q, q_out=q)
    assert got is q and torch.equal(q, apart) and torch.equal(kv, again)
    assert torch.equal(kv[0, :512], c[0]) and torch.equal(kv[cap + 39, :512], c[1]) and torch.equal(kv[2 * cap + 7, :512], c[2])
    assert int((kv != 0).any(1).sum()) == 3


def test_tokens_without_a_place():
    """Past the cap, a negative length, a page outside the pool, a negative page, an offset past the
    cache, tokens that no sequence claims: nothing is written for them, the rest is, and the status
    word says so."""
    cfg = MLAConfig(0, 512, 128, 64, 1, 128)
    g = torch.Generator().manual_seed(5)

    def call(lens, cu, cap, rows, T, **kw):
        kv = torch.zeros(rows, 576, dtype=torch.float16, device=DEV)
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        new = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
        c, k = torch.randn(T, 512, generator=g).half().to(DEV), torch.randn(T, 64, generator=g).half().to(DEV)
        mla_cache_append_rope(kv, c, k, torch.tensor(cu, dtype=torch.int32, device=DEV),
                              torch.tensor(lens, dtype=torch.int32, device=DEV), cap, cfg, new_lens=new, status=st, **kw)
        return sorted((kv != 0).any(1).nonzero()[:, 0].tolist()), int(st), new.tolist()
    assert call([6], [0, 4], 8, 8, 4) == ([6, 7], 1, [8])                       # two of four fit
    assert call([8, 0], [0, 2, 3], 8, 16, 3) == ([8], 1, [8, 1])                 # the first is full
    assert call([-3, 1], [0, 1, 2], 8, 16, 2) == ([9], 1, [-3, 2])
    bad = torch.tensor([[0, 2 ** 31 - 1], [-1, 1]], dtype=torch.int32, device=DEV)
    assert call([63, 62], [0, 2, 5], 128, 128, 5, page_table=bad, page_rows=64) == ([63, 64], 2, [65, 65])
    off = torch.tensor([-1, 15], dtype=torch.int64, device=DEV)
    assert call([0, 0], [0, 2, 4], 8, 16, 4, kv_offsets=off) == ([0, 15], 2, [2, 2])
    assert call([0, 0], [1, 2, 2], 8, 16, 4) == ([0], 1, [1, 0])                 # tokens 0, 2, 3 belong to nobody
    assert call([3, 4], [0, 0, 0], 8, 16, 0) == ([], 0, [3, 4])                  # nothing to append
    assert call([0], [0, 100], 200, 200, 3) == ([0, 1, 2], 0, [3])               # more claimed than given


def test_far_positions():
    """Positions near the end of a 131072-row sequence, whose rows lie past 2^31 bytes of the pool, and
    a row stride: the 64-bit offsets and the exact angles hold."""
    cfg = MLAConfig(0, 512, 128, 64, 2, 128)
    g = torch.Generator().manual_seed(7)
    cap, B = 131072, 16
    pool = torch.empty(B * cap, 640, dtype=torch.bfloat16, device=DEV)
    kv = pool[:, :576]
    c, k = torch.randn(B, 512, generator=g).bfloat16(), torch.randn(B, 64, generator=g).bfloat16()
    lens = [cap - 1 - 1000 * b for b in range(B)]
    mla_cache_append_rope(kv, c.to(DEV), k.to(DEV), torch.arange(B + 1, dtype=torch.int32, device=DEV),
                          torch.tensor(lens, dtype=torch.int32, device=DEV), cap, cfg)
    cos, sin = _tables(cap, 64)
    for b in (0, 7, 15):
        row = kv[b * cap + lens[b]].cpu()
        kd, p = k[b].double(), lens[b]
        want = torch.cat([kd[:32] * cos[p] - kd[32:] * sin[p], kd[:32] * sin[p] + kd[32:] * cos[p]])
        assert torch.equal(row[:512], c[b])
        _near(row[None, 512:], want[None], torch.bfloat16, 8e-7)


def test_another_stream():
    """The call runs on the current stream, behind what made its inputs there."""
    cfg = MLAConfig(0, 512, 128, 64, 16, 128)
    side = torch.cuda.Stream()
    x = torch.randn(64, 512, device=DEV).bfloat16()
    k = torch.randn(64, 64, device=DEV).bfloat16()
    cu, lens = torch.tensor([0, 64], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    kv = torch.zeros(64, 576, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = x + 1
        mla_cache_append_rope(kv, y, k, cu, lens, 64, cfg)
    side.synchronize()
    assert torch.equal(kv[:, :512], x + 1)


def test_refusals():
    cfg = MLAConfig(0, 512, 128, 64, 4, 128)
    kv = torch.zeros(64, 576, dtype=torch.bfloat16, device=DEV)
    c, k = torch.zeros(2, 512, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    cu, lens = torch.tensor([0, 2], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)

    def refuses(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            mla_cache_append_rope(*a, cfg, **kw)
    refuses("c must be", kv, c.half(), k, cu, lens, 64)
    refuses("k_rope must be", kv, c, k[:1], cu, lens, 64)
    refuses("unit inner stride", kv, torch.zeros(512, 2, dtype=torch.bfloat16, device=DEV).t(), k, cu, lens, 64)
    refuses("cu_tokens", kv, c, k, cu[:1], lens, 64)
    refuses("cu_tokens", kv, c, k, cu.long(), lens, 64)
    refuses("kv_cache", kv[:, :575], c, k, cu, lens, 64)
    refuses("max_seq_len", kv, c, k, cu, lens, 0)
    refuses("both rope_cos", kv, c, k, cu, lens, 64, rope_cos=torch.zeros(64, 32, device=DEV))
    refuses("rope_cos must be", kv, c, k, cu, lens, 64, rope_cos=torch.zeros(63, 32, device=DEV),
            rope_sin=torch.zeros(63, 32, device=DEV))
    refuses("seq_lens", kv, c, k, cu, lens, 64, new_lens=lens)
    refuses("q_out needs", kv, c, k, cu, lens, 64, q_out=q)
    refuses("overlap", kv, c, k, cu, lens, 64, q_rope=q, q_out=q[:1].expand(2, 4, 64))
    refuses("page_rows", kv, c, k, cu, lens, 64, page_table=torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    refuses("max_pages", kv, c, k, cu, lens, 65, page_table=torch.zeros(1, 1, dtype=torch.int32, device=DEV), page_rows=64)
    refuses("excludes", kv, c, k, cu, lens, 64, page_table=torch.zeros(1, 1, dtype=torch.int32, device=DEV),
            page_rows=64, kv_offsets=torch.zeros(1, dtype=torch.int64, device=DEV))
    refuses("norm_eps", kv, c, k, cu, lens, 64, norm_weight=torch.zeros(512, dtype=torch.bfloat16, device=DEV),
            norm_eps=-1.0)
    assert int(kv.abs().sum()) == 0


def test_a_cache_whose_rows_overlap_is_refused():
    cfg = MLAConfig(0, 512, 128, 64, 4, 128)
    row = torch.zeros(1, 576, dtype=torch.bfloat16, device=DEV)
    c, k = torch.ones(2, 512, dtype=torch.bfloat16, device=DEV), torch.ones(2, 64, dtype=torch.bfloat16, device=DEV)
    cu, lens = torch.tensor([0, 2], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        mla_cache_append_rope(row.expand(64, 576), c, k, cu, lens, 64, cfg)
    assert int(row.abs().sum()) == 0
    one = row.view(-1).as_strided((1, 576), (0, 1))               # a single row has any stride
    mla_cache_append_rope(one, c[:1], k[:1], cu - torch.tensor([0, 1], dtype=torch.int32, device=DEV), lens, 1, cfg)
    assert torch.equal(row[0, :512], c[0])


@pytest.mark.parametrize("T,H", [(5, 4), (1, 4), (5, 1), (1, 1)])
def test_queries_with_heads_outside_tokens(T, H):
    """Inputs and outputs laid out (H, T, d_R), with and without gaps, give the bits of the contiguous form."""
    cfg = MLAConfig(0, 512, 128, 64, H, 128)
    g = torch.Generator().manual_seed(T + H)
    c, k, q = [torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV) for shape in ((T, 512), (T, 64), (T, H, 64))]
    cu, lens = torch.tensor([0, T], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)

    def call(**kw):
        kv = torch.zeros(64, 576, dtype=torch.bfloat16, device=DEV)
        return mla_cache_append_rope(kv, c, k, cu, lens, 64, cfg, **kw)
    want = call(q_rope=q)
    for gap in (0, 8):
        wide = torch.full((H, T, 64 + gap), 7.0, dtype=torch.bfloat16, device=DEV)
        out = wide.permute(1, 0, 2)[..., :64]
        src = torch.zeros(H, T, 64 + gap, dtype=torch.bfloat16, device=DEV).permute(1, 0, 2)[..., :64]
        src.copy_(q)
        assert torch.equal(call(q_rope=src, q_out=out), want) and (wide[..., 64:] == 7).all()
        assert torch.equal(call(q_rope=src, q_out=src), want)      # in place
    flat = torch.zeros(T * H * 64 + 64, dtype=torch.bfloat16, device=DEV)
    for strides in ((64 * H, 63, 1), (63, 64 * T, 1), (64, 64, 1)):
        if (H > 1 and strides[1] < 64) or (T > 1 and (strides[0] < 64 or (H > 1 and strides[0] == strides[1]))):
            with pytest.raises(RuntimeError, match="overlap"):
                call(q_rope=q, q_out=flat.as_strided((T, H, 64), strides))
