"""The layer's serving step (prefix_decode_step): projections with adapters, append with norm and
rotation, attention over shared prefixes, value and output projections, against the same formulas
in float64 with the kernels' 16-bit weights and inputs.

Tolerance: the chain rounds to 16 bits at the queries, the cache rows, the latent output, the value
projection and the result, each by 2^-9 of its size in bf16 at most; the queries' rounding moves a
score of size s by about s 2^-9 sqrt(2), and with |s| <= 8 a softmax weight by less than 1 percent of
itself in one direction for some and in the other for the rest. Hence the suite's decode bound:
max|d| / max|ref| <= 2e-2 and cosine > 0.998."""

import math

import numpy as np
import pytest
import torch

from oracle import mla_oracle as O
from latent_attn import LatentAttentionLayer, MLAConfig, SharedPrefixBatch, functional

pytestmark = pytest.mark.gpu

MAX_REL, MIN_COS = 2e-2, 0.998
H, DC, DR, DV, DM, RANK, NA = 16, 512, 64, 128, 512, 16, 3
SIZES, PREFIX, OWN = [3, 1, 2], [128, 0, 192], [0, 5, 64, 0, 63, 1]
CAP = 70
EPS = 1e-6


def _layer():
    torch.manual_seed(11)
    cfg = MLAConfig(DM, DC, 128, DR, H, DV)
    return LatentAttentionLayer(cfg, 512).cuda(), cfg


def _rot(x, p):
    cos, sin = O.rope_tables(1, x.shape[-1], pos_offset=int(p))
    h = x.shape[-1] // 2
    return np.concatenate([x[..., :h] * cos[0] - x[..., h:] * sin[0], x[..., :h] * sin[0] + x[..., h:] * cos[0]], -1)


def _row(c, k, w, p):
    return np.concatenate([c / math.sqrt((c * c).mean() + EPS) * w, _rot(k, p)])


def _f64(t):
    return t.detach().cpu().double().numpy()


def _want(layer, dt, x, rows, p, adapter):
    """One token: x (DM,), all its rows in order, its position, its adapters per projection or None."""
    w = {n: _f64(getattr(layer, n).to(dt)) for n in ("W_Q_absorbed", "W_Q_rope", "W_UV", "W_O")}

    def project(name, v):
        y = w[name] @ v
        if adapter is not None and name in adapter:
            a, b, s = adapter[name]
            y = y + s * (b @ (a @ v))
        return y

    qa = project("W_Q_absorbed", x).reshape(H, DC)
    qr = _rot(project("W_Q_rope", x).reshape(H, DR), p)
    s = (qa @ rows[:, :DC].T + qr @ rows[:, DC:].T) / math.sqrt(128 + DR)
    e = np.exp(s - s.max(1, keepdims=True))
    o = (e / e.sum(1, keepdims=True)) @ rows[:, :DC]
    v = np.einsum("hc,hjc->hj", o, w["W_UV"].reshape(H, DV, DC))
    return project("W_O", v.reshape(-1))


@pytest.mark.parametrize("adapters", [False, True])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_steps(dt, paged, adapters):
    layer, cfg = _layer()
    g = torch.Generator().manual_seed(12)
    B = sum(SIZES)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dt)

    first = [n for n, size in zip(PREFIX, SIZES) for _ in range(size)]
    norm_w = rnd(DC).abs() + 0.5
    pc, pk = rnd(sum(PREFIX), DC), rnd(sum(PREFIX), DR)          # the prefixes' tokens
    oc, ok = rnd(sum(OWN), DC), rnd(sum(OWN), DR)                # the requests' tokens so far
    ids = torch.tensor([0, 2, -1, 2, 1, 0], dtype=torch.int32)
    ad = {n: (rnd(NA, RANK, k, scale=k ** -0.5), rnd(NA, o, RANK, scale=0.1), torch.tensor([0.5, 1.0, 2.0]))
          for n, k, o in (("W_Q_absorbed", DM, H * DC), ("W_O", H * DV, DM))} if adapters else None

    # where the rows lie, and the rows that are there before the first step
    if paged:
        R = 64
        order = torch.randperm(40, generator=g).tolist()
        ptab = [[order.pop() for _ in range(3)] for _ in PREFIX]
        otab = [[order.pop() for _ in range(2)] for _ in range(B)]
        batch = SharedPrefixBatch(cfg, "cuda", SIZES, PREFIX, OWN, CAP, prefix_table=ptab, own_table=otab, page_rows=R)
        kv = torch.full((40 * R, DC + DR), float("nan"), dtype=dt, device="cuda")
    else:
        poff = [3, 140, 200]
        ooff = [400 + (CAP + 2) * b for b in range(B)]
        batch = SharedPrefixBatch(cfg, "cuda", SIZES, PREFIX, OWN, CAP, prefix_offsets=poff, own_offsets=ooff)
        kv = torch.full((1000, DC + DR), float("nan"), dtype=dt, device="cuda")

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def cum(v):
        return i32([0] + np.cumsum(v).tolist())

    tables = {"rope_cos": layer.rope_cos, "rope_sin": layer.rope_sin, "norm_weight": norm_w.cuda(), "norm_eps": EPS}
    functional.mla_cache_append_rope(kv, pc.cuda(), pk.cuda(), cum(PREFIX), i32([0] * len(PREFIX)), batch.max_prefix_len, cfg,
                                     kv_offsets=batch.prefix_offsets, page_table=batch.prefix_table,
                                     page_rows=batch.page_rows, **tables)
    functional.mla_cache_append_rope(kv, oc.cuda(), ok.cuda(), cum(OWN), i32(first), batch.max_positions, cfg,
                                     kv_offsets=batch.row_offsets, page_table=batch.row_table,
                                     page_rows=batch.page_rows, **tables)
    w = _f64(norm_w)
    pstart, ostart = np.cumsum([0] + PREFIX), np.cumsum([0] + OWN)
    prefix_rows = [[_row(_f64(pc[pstart[q] + i]), _f64(pk[pstart[q] + i]), w, i) for i in range(PREFIX[q])]
                   for q in range(len(PREFIX))]
    group = [q for q, size in enumerate(SIZES) for _ in range(size)]
    rows = [prefix_rows[group[b]] + [_row(_f64(oc[ostart[b] + i]), _f64(ok[ostart[b] + i]), w, first[b] + i)
                                     for i in range(OWN[b])] for b in range(B)]

    dev_ad = None if ad is None else {n: tuple(t.cuda() for t in v) for n, v in ad.items()}
    for step in range(3):
        x, c, k = rnd(B, DM), rnd(B, DC), rnd(B, DR)
        got = layer.prefix_decode_step(x.cuda(), c.cuda(), k.cuda(), kv, batch, norm_weight=norm_w.cuda(), norm_eps=EPS,
                                       adapters=dev_ad, adapter_ids=None if ad is None else ids.cuda())
        assert got.shape == (B, DM) and got.dtype == dt
        want = []
        for b in range(B):
            p = first[b] + OWN[b] + step
            rows[b].append(_row(_f64(c[b]), _f64(k[b]), w, p))
            a = int(ids[b])
            own = None if ad is None or a < 0 else {n: (_f64(v[0][a]), _f64(v[1][a]), float(v[2][a])) for n, v in ad.items()}
            want.append(_want(layer, dt, _f64(x[b]), np.array(rows[b]), p, own))
        cmp = O.compare(_f64(got), np.array(want))
        assert cmp["finite"] and cmp["max_rel"] <= MAX_REL and cmp["cosine"] > MIN_COS, (step, cmp)
        assert batch.own_lens.tolist() == [n + step + 1 for n in OWN]


def test_refusals():
    layer, cfg = _layer()
    kv = torch.zeros(64, DC + DR, dtype=torch.bfloat16, device="cuda")
    batch = SharedPrefixBatch(cfg, "cuda", [1], [8], [3], 4, prefix_offsets=[0], own_offsets=[8])
    x, c, k = torch.zeros(1, DM, device="cuda"), torch.zeros(1, DC, device="cuda"), torch.zeros(1, DR, device="cuda")
    with pytest.raises(RuntimeError, match="adapter_ids"):
        layer.prefix_decode_step(x, c, k, kv, batch, adapters={"W_O": None})
    with pytest.raises(RuntimeError, match="x must be"):
        layer.prefix_decode_step(x[:, :8], c, k, kv, batch)
    layer.prefix_decode_step(x, c, k, kv, batch)
    with pytest.raises(RuntimeError, match="max_own_len"):
        layer.prefix_decode_step(x, c, k, kv, batch)


@pytest.mark.parametrize("paged", [False, True])
def test_a_captured_step_advances(paged):
    """Replays of one captured step write the rows of eager steps to the bit, and give their outputs, until a
    request is full; then its token is dropped, its lengths and every row stay, and the batch's status says so.

    The outputs pass mla_linear, whose fp32 sums over a split K may differ in their last bits from call to call:
    by 2^-18 of the largest output at most, and then by a step of bf16 (2^-7 of the value)."""
    layer, cfg = _layer()
    dt, B, steps = torch.bfloat16, sum(SIZES), 4
    own = [0, 5, 64, 1, 63, 1]
    cap = max(own) + steps
    g = torch.Generator().manual_seed(31)

    def batch_and_cache():
        kv = torch.randn(64 * 40, DC + DR, generator=torch.Generator().manual_seed(32)).to(dt).cuda()
        if paged:
            order = torch.randperm(40, generator=torch.Generator().manual_seed(33)).tolist()
            where = dict(prefix_table=[[order.pop() for _ in range(3)] for _ in PREFIX],
                         own_table=[[order.pop() for _ in range(2)] for _ in range(B)], page_rows=64)
        else:
            where = dict(prefix_offsets=[3, 140, 200], own_offsets=[400 + cap * b for b in range(B)])
        return SharedPrefixBatch(cfg, "cuda", SIZES, PREFIX, own, cap, **where), kv

    data = [[torch.randn(B, n, generator=g).to(dt).cuda() for n in (DM, DC, DR)] for _ in range(steps)]
    eager, kv = batch_and_cache()
    want = []
    for x, c, k in data:
        y = layer.prefix_decode_step(x, c, k, kv, eager)
        want.append((y, kv.clone(), eager.own_lens.tolist()))
    assert int(eager.status) == 0
    with pytest.raises(RuntimeError, match="max_own_len"):
        layer.prefix_decode_step(*data[0], kv, eager)

    batch, kv = batch_and_cache()
    held = [t.clone() for t in data[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.prefix_decode_step(*held, kv, batch)
    for i in range(steps):
        for h, t in zip(held, data[i]):
            h.copy_(t)
        graph.replay()
        y, rows, lens = want[i]
        assert batch.own_lens.tolist() == lens
        assert torch.equal(kv, rows), i
        assert bool(((out - y).abs() <= 2.0 ** -7 * y.abs() + 2.0 ** -18 * y.abs().max()).all()), i
    assert int(batch.status) == 0
    # the third request is full: only its rows stay as they are
    before, full = kv.clone(), batch.own_lens.tolist()
    graph.replay()
    graph.replay()
    assert int(batch.status) & 1
    assert batch.own_lens.tolist() == [min(n + 2, cap) for n in full]
    changed = set((kv != before).any(1).nonzero()[:, 0].tolist())
    expect = set()
    for b, n in enumerate(full):
        for i in range(n, min(n + 2, cap)):
            expect.add(int(batch.own_table[b, i // 64]) * 64 + i % 64 if paged else int(batch.own_offsets[b]) + i)
    assert changed == expect
