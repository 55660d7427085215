"""mla_prefix_decode against its definition in 64 bits: shared prefixes of one to several groups,
requests with and without rows of their own, both layouts, head counts that fill, straddle and
underfill a 128-row tile, lengths around the 64-row tile, and what lies past a sequence's end.

Tolerance. The inputs are 16-bit values that the oracle reads as they are. What a kernel may add:
P rounded to the cache's type (u = 2^-8 for bf16, 2^-11 for fp16, at most u relative on each
weight), partial scores exchanged in fp16 (2^-11 of a partial, whose size here is below 16 in log2
units: below 2^-7 in the exponent, 0.0055 relative on each weight), a partial record and the result
rounded to the cache's type (u each). Each of these errors is independent from element to element,
so the norm of the difference is far below the sum of the bounds; the test allows the root of the
sum of their squares: bf16 sqrt(3 u^2 + 0.0055^2) = 8.7e-3, fp16 5.6e-3 of an output row's norm,
and 8 times that of the row's root mean square for any single element (512 of them)."""

import math

import pytest
import torch

from latent_attn import MLAConfig, _lib
from latent_attn.functional import mla_prefix_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 1.0 / math.sqrt(192)
AUTO, TC, SIMT = 0, 1, 2


class Case:
    """Inputs of one call, and the rows that each request attends to."""

    def __init__(self, sizes, prefix, own, heads, dtype, page=0, dc=512, dR=64, seed=0, poison=None, gap=5):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.prefix, self.own, self.heads, self.dtype, self.dc, self.dR = sizes, prefix, own, heads, dtype, dc, dR
        B, self.page = sum(sizes), page
        lens = list(prefix) + list(own)
        self.rows_of, at = [], gap
        if page:
            need = [-(-n // page) for n in lens]
            ids = torch.randperm(sum(need) + 3, generator=g)
            total = (sum(need) + 3) * page
            table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
            k = 0
            for i, n in enumerate(need):
                table[i, :n] = ids[k:k + n].to(torch.int32)
                k += n
                p = torch.arange(lens[i])
                self.rows_of.append(table[i].long()[p // page] * page + p % page)
            self.ptable, self.table = table[:len(prefix)].contiguous(), table[len(prefix):].contiguous()
        else:
            for n in lens:
                self.rows_of.append(torch.arange(at, at + n))
                at += n + gap
            total = at
        kv = torch.randn(total, dc + dR, generator=g)
        if poison is not None:                                   # every row that nobody attends to
            used = torch.zeros(total, dtype=torch.bool)
            for r in self.rows_of:
                used[r] = True
            kv[~used] = poison
        self.kv = kv.to(dtype)
        self.qa = (0.5 * torch.randn(B, heads, dc, generator=g) * math.sqrt(512 / dc)).to(dtype)
        self.qr = torch.randn(B, heads, dR, generator=g).to(dtype)
        self.starts = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32)

    def args(self, **over):
        kw = dict(group_starts=self.starts.to(DEV), prefix_lens=torch.tensor(self.prefix, dtype=torch.int32, device=DEV),
                  max_prefix_len=max(self.prefix), seq_lens=torch.tensor(self.own, dtype=torch.int32, device=DEV),
                  max_seq_len=max(self.own), page_rows=self.page, softmax_scale=SCALE)
        if self.page:
            kw.update(prefix_table=self.ptable.to(DEV), page_table=self.table.to(DEV))
        else:
            n = len(self.prefix)
            first = [int(r[0]) if len(r) else 0 for r in self.rows_of]
            kw.update(prefix_offsets=torch.tensor(first[:n], dtype=torch.int64, device=DEV),
                      kv_offsets=torch.tensor(first[n:], dtype=torch.int64, device=DEV))
        kw.update(over)
        return kw

    def run(self, kernel=AUTO, **over):
        cfg = MLAConfig(0, self.dc, 128, self.dR, self.heads, 128)
        return mla_prefix_decode(self.kv.to(DEV), self.qa.to(DEV), self.qr.to(DEV), cfg, kernel=kernel, **self.args(**over))

    def exact(self):
        kv, out, b = self.kv.to(DEV).double(), [], 0
        for g, n in enumerate(self.sizes):
            for _ in range(n):
                rows = torch.cat([self.rows_of[g], self.rows_of[len(self.sizes) + b]]).to(DEV)
                k = kv[rows]
                s = (self.qa[b].to(DEV).double() @ k[:, :self.dc].T + self.qr[b].to(DEV).double() @ k[:, self.dc:].T) * SCALE
                p = torch.softmax(s, -1) if len(rows) else s
                out.append(p @ k[:, :self.dc])
                b += 1
        return torch.stack(out)


def check(got, want, dtype, what=""):
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    tol = math.sqrt(3 * u * u + 0.0055 ** 2)
    assert got.dtype == dtype and torch.isfinite(got).all(), what
    d, norm = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    assert bool((d <= tol * norm).all()), (what, float((d / norm.clamp(min=1e-30)).max()))
    big = (got.double() - want).abs().amax(-1)
    assert bool((big <= 8 * tol * norm / math.sqrt(want.shape[-1])).all()), (what, "one element")


KERNELS = [AUTO, SIMT]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 16, 24, 128])
@pytest.mark.parametrize("page", [0, 64, 192])
def test_groups(kernel, dtype, heads, page):
    """Three groups (one of a single request, one without a prefix), own lengths from nothing on."""
    c = Case([5, 1, 4], [300, 65, 0], [0, 1, 63, 64, 65, 200, 7, 128, 1, 130], heads, dtype, page, seed=heads + page)
    check(c.run(kernel), c.exact(), dtype)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 1000])
def test_prefix_lengths(kernel, n):
    c = Case([9], [n], [0] * 9, 16, torch.bfloat16, 64, seed=n)
    check(c.run(kernel), c.exact(), torch.bfloat16, n)


@pytest.mark.parametrize("heads,batch", [(3, 43), (48, 9), (96, 4), (130, 3), (256, 2), (64, 33)])
def test_head_layouts(heads, batch):
    """Rows of several requests in one tile, tiles that straddle requests, more than 128 heads."""
    own = [(37 * b) % 150 for b in range(batch)]
    c = Case([batch - 1, 1], [500, 77], own, heads, torch.bfloat16, 0, seed=heads)
    check(c.run(), c.exact(), torch.bfloat16)


@pytest.mark.parametrize("kernel", KERNELS)
def test_empty_rows_give_zero(kernel):
    c = Case([2, 2], [0, 70], [0, 5, 0, 3], 16, torch.bfloat16, 64)
    out = c.run(kernel)
    assert int((out[0] != 0).sum()) == 0
    check(out[1:], c.exact()[1:], torch.bfloat16)
    none = Case([3], [0], [0, 0, 0], 16, torch.bfloat16, 64)
    assert int((none.run(kernel) != 0).sum()) == 0               # maximum lengths of zero


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_rows_past_the_end_do_not_count(kernel, page, poison):
    """Whatever lies in the rows past a length, in the same page or tile, stays out."""
    c = Case([3, 2], [100, 1], [1, 70, 0, 33, 64], 16, torch.bfloat16, page, poison=poison)
    check(c.run(kernel), c.exact(), torch.bfloat16)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_stays_with_its_requests(kernel):
    c = Case([2, 2], [100, 100], [10, 10, 10, 10], 16, torch.bfloat16, 64)
    c.kv[c.rows_of[1][5], 3] = math.nan                           # the second group's prefix
    c.kv[c.rows_of[2][5], 3] = math.nan                           # the first request's own rows
    out = c.run(kernel)
    assert torch.isnan(out[0]).any() and torch.isnan(out[2]).any() and torch.isnan(out[3]).any()
    check(out[1:2], c.exact()[1:2], torch.bfloat16)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rising_and_falling_scores(kernel, dtype):
    """A running maximum that keeps moving (by more than any rescaling threshold), across prefix, own
    rows and workers, and rows whose first tiles count for nothing."""
    c = Case([8], [3000], [200, 0, 64, 1, 500, 90, 3, 1000], 16, dtype, 64, seed=11)
    q = c.qa[:, :, :].float().mean(1, keepdim=True)
    for i, r in enumerate([c.rows_of[0]] + c.rows_of[1:]):
        ramp = torch.linspace(-3, 3, max(len(r), 1))[:len(r)] * (1 if i % 2 == 0 else -1)
        c.kv[r, 0] = ramp.to(dtype) * 3
    c.qa[:, :, 0] = 8.0
    check(c.run(kernel), c.exact(), dtype)


def test_long_prefix_and_many_workers():
    c = Case([6], [50000], [0, 1, 100, 2000, 64, 5], 16, torch.bfloat16, 128, seed=5)
    check(c.run(), c.exact(), torch.bfloat16)


def test_lengths_above_the_bound_are_cut():
    c = Case([3], [200], [90, 10, 70], 16, torch.bfloat16, 64)
    cut = Case([3], [200], [90, 10, 70], 16, torch.bfloat16, 64)
    cut.rows_of[0] = cut.rows_of[0][:130]
    cut.rows_of[1:] = [r[:65] for r in cut.rows_of[1:]]
    check(c.run(max_prefix_len=130, max_seq_len=65), cut.exact(), torch.bfloat16)


@pytest.mark.parametrize("kernel", KERNELS)
def test_requests_outside_every_group(kernel):
    c = Case([4], [100], [10, 20, 30, 40], 16, torch.bfloat16, 64)
    want = c.exact()
    out = c.run(kernel, group_starts=torch.tensor([1, 3], dtype=torch.int32, device=DEV))
    check(out[1:3], want[1:3], torch.bfloat16)
    alone = Case([4], [0], [10, 20, 30, 40], 16, torch.bfloat16, 64)
    alone.kv, alone.qa, alone.qr, alone.rows_of = c.kv, c.qa, c.qr, [c.rows_of[0][:0]] + c.rows_of[1:]
    check(out[[0, 3]], alone.exact()[[0, 3]], torch.bfloat16)


@pytest.mark.parametrize("kernel", KERNELS)
def test_bad_pages_and_offsets_read_nothing(kernel):
    c = Case([3, 1], [130, 64], [70, 10, 70, 70], 16, torch.bfloat16, 64)
    t = c.table.clone()
    t[0, 1], t[2, 0] = 1 << 20, -5
    out = c.run(kernel, page_table=t.to(DEV))
    assert torch.isnan(out[0]).all() and torch.isnan(out[2]).all()
    check(out[[1, 3]], c.exact()[[1, 3]], torch.bfloat16)
    d = Case([2], [64], [5, 5], 16, torch.bfloat16, 0)
    out = d.run(kernel, kv_offsets=torch.tensor([-3, int(d.rows_of[2][0])], dtype=torch.int64, device=DEV))
    assert torch.isnan(out[0]).all()
    check(out[1:], d.exact()[1:], torch.bfloat16)


def test_row_stride_and_far_rows():
    """Rows of a wider pool, whose byte offsets pass 2^32."""
    c = Case([3], [150], [10, 0, 64], 16, torch.bfloat16, 64, seed=9)
    want = c.exact()
    rows, far = c.kv.shape[0], 3_600_000
    pool = torch.empty(far + rows, 640, dtype=torch.bfloat16, device=DEV)
    pool[far:, :576] = c.kv.to(DEV)
    assert far % 64 == 0
    cfg = MLAConfig(0, 512, 128, 64, 16, 128)
    shift = far // 64
    kw = c.args(prefix_table=torch.where(c.ptable >= 0, c.ptable + shift, -1).to(DEV),
                page_table=torch.where(c.table >= 0, c.table + shift, -1).to(DEV))
    for kernel in KERNELS:
        check(mla_prefix_decode(pool[:, :576], c.qa.to(DEV), c.qr.to(DEV), cfg, kernel=kernel, **kw), want, torch.bfloat16)


@pytest.mark.parametrize("dc,dR", [(256, 64), (96, 16), (1024, 128), (512, 30)])
def test_other_widths(dc, dR):
    c = Case([3, 2], [90, 130], [0, 64, 3, 10, 1], 8, torch.float16, 64, dc=dc, dR=dR)
    check(c.run(), c.exact(), torch.float16)


def test_same_result_every_time_and_on_a_side_stream():
    c = Case([16, 8], [2000, 777], [(53 * b) % 300 for b in range(24)], 16, torch.bfloat16, 64)
    first = c.run()
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)   # an uninitialised workspace
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = [c.run(workspace=ws) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(first, a) for a in again)


def test_in_a_cuda_graph():
    c = Case([4, 3], [500, 40], [9, 0, 64, 65, 1, 200, 70], 16, torch.bfloat16, 64)
    cfg = MLAConfig(0, 512, 128, 64, 16, 128)
    kv, qa, qr, kw = c.kv.to(DEV), c.qa.to(DEV), c.qr.to(DEV), c.args()
    call = lambda: mla_prefix_decode(kv, qa, qr, cfg, **kw)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    kw["seq_lens"].copy_(torch.tensor([3, 0, 1, 65, 1, 100, 0], dtype=torch.int32))   # new lengths, same graph
    graph.replay()
    c.rows_of[2:] = [r[:n] for r, n in zip(c.rows_of[2:], [3, 0, 1, 65, 1, 100, 0])]
    check(out, c.exact(), torch.bfloat16)


def test_refusals():
    c = Case([2], [64], [5, 5], 16, torch.bfloat16, 64)

    def refuses(match, **over):
        with pytest.raises(RuntimeError, match=match):
            c.run(**over)
    refuses("multiple of 64", page_rows=32)
    refuses("excludes", kv_offsets=torch.zeros(2, dtype=torch.int64, device=DEV))
    refuses("fewer pages", max_seq_len=65)
    refuses("fewer pages", max_prefix_len=65)
    refuses("needs prefix_table", page_table=None)
    refuses("page tables need", page_rows=0)
    refuses("group_starts", group_starts=torch.zeros(2, dtype=torch.int64, device=DEV))
    refuses("seq_lens", seq_lens=torch.zeros(3, dtype=torch.int32, device=DEV))
    refuses("softmax_scale", softmax_scale=-1.0)
    refuses("softmax_scale", softmax_scale=math.nan)
    refuses("out must be", out=torch.empty(2, 16, 512, device=DEV))
    refuses("unknown kernel", kernel=7)
    cfg = MLAConfig(0, 512, 128, 64, 16, 128)
    with pytest.raises(RuntimeError, match="q_rope must be"):
        mla_prefix_decode(c.kv.to(DEV), c.qa.to(DEV), c.qr.to(DEV).half(), cfg, **c.args())
    with pytest.raises(RuntimeError, match="contiguous"):
        mla_prefix_decode(c.kv.to(DEV), c.qa.to(DEV).transpose(0, 1).contiguous().transpose(0, 1), c.qr.to(DEV), cfg, **c.args())
    with pytest.raises(RuntimeError, match="kv_cache"):
        mla_prefix_decode(c.kv.to(DEV)[:, :570], c.qa.to(DEV), c.qr.to(DEV), cfg, **c.args())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("starts", [[0, 64] * 32, [0, 5, 3, 64], [64, 0], [0, 1 << 30, -(1 << 30), 64],
                                    [0, 64] * 700])
def test_decreasing_group_starts(kernel, heads, starts, monkeypatch):
    """Ranges of requests that overlap: NaN everywhere, and nothing outside the workspace or the output. Each
    pair of [0, 64] alone has as many row groups as the workspace has for all requests."""
    P = len(starts) - 1
    g = torch.Generator().manual_seed(heads)
    kv = torch.randn(1024, 576, generator=g).to(torch.bfloat16).to(DEV)
    qa = torch.randn(64, heads, 512, generator=g).to(torch.bfloat16).to(DEV)
    qr = torch.randn(64, heads, 64, generator=g).to(torch.bfloat16).to(DEV)
    kw = dict(prefix_lens=torch.full((P,), 130, dtype=torch.int32, device=DEV), max_prefix_len=130,
              seq_lens=torch.arange(64, dtype=torch.int32, device=DEV), max_seq_len=64,
              prefix_offsets=torch.zeros(P, dtype=torch.int64, device=DEV),
              kv_offsets=torch.arange(64, device=DEV) * 8, kernel=kernel)
    cfg = MLAConfig(0, 512, 128, 64, heads, 128)
    packed, need = _lib.load_packed(), []
    real = packed.mla_prefix_decode
    monkeypatch.setattr(packed, "mla_prefix_decode", lambda *a: need.append(a[3]) or real(*a))
    ws = torch.full((192 << 20,), 0xA5, dtype=torch.uint8, device=DEV)
    wide = torch.full((3, 64, heads, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    mla_prefix_decode(kv, qa, qr, cfg, group_starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                      out=wide[1], workspace=ws, **kw)
    assert torch.isnan(wide[1]).all() and (wide[0] == 7).all() and (wide[2] == 7).all()
    assert need[0] < ws.numel() and (ws[need[0]:] == 0xA5).all()
    # the same workspace serves a proper call after it
    want = mla_prefix_decode(kv, qa, qr, cfg, group_starts=torch.tensor(sorted(starts), dtype=torch.int32, device=DEV), **kw)
    got = mla_prefix_decode(kv, qa, qr, cfg, group_starts=torch.tensor(sorted(starts), dtype=torch.int32, device=DEV),
                            workspace=ws, **kw)
    assert torch.isfinite(got).all() and torch.equal(got, want)


def test_workspaces_that_the_kernels_cannot_write_are_refused():
    c = Case([2], [64], [5, 5], 16, torch.bfloat16, 64)
    for ws in (torch.empty(64 << 20, dtype=torch.uint8), torch.empty(64 << 20, dtype=torch.uint8).pin_memory(),
               torch.empty(1, dtype=torch.uint8, device=DEV).expand(64 << 20)):
        for kernel in KERNELS:
            with pytest.raises(RuntimeError, match="workspace must be"):
                c.run(kernel, workspace=ws)
    check(c.run(workspace=torch.empty(1, dtype=torch.uint8, device=DEV)), c.exact(), torch.bfloat16)


def test_a_cache_whose_rows_overlap_is_refused():
    c = Case([2], [64], [5, 5], 16, torch.bfloat16, 64)
    cfg = MLAConfig(0, 512, 128, 64, 16, 128)
    row = torch.ones(1, 576, dtype=torch.bfloat16, device=DEV)
    for kv in (row.expand(640, 576), row.view(-1).as_strided((2, 576), (0, 1)), row.expand(4, 576).reshape(-1).as_strided((4, 576), (570, 1))):
        for kernel in KERNELS:
            with pytest.raises(RuntimeError, match="overlap"):
                mla_prefix_decode(kv, c.qa.to(DEV), c.qr.to(DEV), cfg, kernel=kernel, **c.args())
    # a single row has any stride
    one = Case([1], [0], [1], 16, torch.bfloat16, 0, gap=0)
    kv = one.kv.to(DEV).as_strided((1, 576), (0, 1))
    got = mla_prefix_decode(kv, one.qa.to(DEV), one.qr.to(DEV), cfg, **one.args())
    check(got, one.exact(), torch.bfloat16)


# Scores of any size. The tolerance does not grow with them: a score of up to 2^10 (log2 units) is a sum in
# fp32, whose 18 steps of 16 products each round to 2^-14 at that size (a standard deviation below 2^-12), and
# whose two halves may each be rounded by 2^-22 of the row's largest, 2^-12: together below 2^-11 in the
# exponent as a standard deviation of several. P, the records and the result are rounded as above (u each):
# bf16 sqrt(3 u^2 + 2^-22) = 6.8e-3 of a row's norm, fp16 9.8e-4, 8 times that for one element.
def check_any_size(got, want, what=""):
    u = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    tol = math.sqrt(3 * u * u + 2.0 ** -22)
    assert torch.isfinite(got).all(), what
    d, norm = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    assert bool((d <= tol * norm).all()), (what, float((d / norm.clamp(min=1e-30)).max()), tol)
    big = (got.double() - want).abs().amax(-1)
    assert bool((big <= 8 * tol * norm / math.sqrt(want.shape[-1])).all()), (what, "one element")


def _sized(heads, dtype, seed):
    return Case([6, 3], [700, 130], [0, 1, 65, 300, 40, 64, 5, 128, 200], heads, dtype, 64, seed=seed)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("size", [4.0, 30.0, 100.0])
def test_sharp_scores(size, heads, dtype, kernel):
    """Scores whose standard deviation is `size` / 3 (most within +-size), and so single keys that decide."""
    c = _sized(heads, dtype, seed=21)
    c.qa, c.qr = (c.qa.float() * size / 3).to(dtype), (c.qr.float() * size / 3).to(dtype)
    check_any_size(c.run(kernel), c.exact(), (size, heads))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("offset", [-600.0, -64.0, 64.0, 500.0])
@pytest.mark.parametrize("column", [0, 40])
def test_an_offset_common_to_all_keys(column, offset, heads, dtype, kernel):
    """A large constant in every score (softmax does not see it), from either half of the columns."""
    c = _sized(heads, dtype, seed=22)
    c.kv[:, 512 + column] = 8.0
    c.qr[..., column] = offset / (8.0 * SCALE)
    check_any_size(c.run(kernel), c.exact(), (column, offset, heads))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("size", [30.0, 100.0, 600.0])
def test_halves_that_cancel(size, heads, dtype, kernel):
    """Every key has a part of its score of up to +-size in one half of the columns and its opposite in the
    other (the products are exact, so nothing of it is left in the sum)."""
    c = _sized(heads, dtype, seed=23)
    g = torch.Generator().manual_seed(24)
    part = torch.randint(-8, 9, (c.kv.shape[0],), generator=g).to(dtype)
    c.kv[:, 512 + 3], c.kv[:, 512 + 35] = part, part
    c.qr[..., 3] = size / (8.0 * SCALE)
    c.qr[..., 35] = -c.qr[..., 3]
    check_any_size(c.run(kernel), c.exact(), (size, heads))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", ["lowest", "-inf"])
def test_keys_masked_by_the_lowest_value(value, dtype, kernel):
    """Keys with the type's lowest value or -inf in a column where every query has 1: their weight is zero, the
    others' as without them; and where all keys have the lowest value, none is preferred for it."""
    c = _sized(16, dtype, seed=25)
    c.qr[..., 7] = 1.0
    c.kv[:, 512 + 7] = 0.0
    masked = torch.zeros(c.kv.shape[0], dtype=torch.bool)
    for r in c.rows_of:
        masked[r[1::3]] = True
    low = torch.finfo(dtype).min if value == "lowest" else -math.inf
    c.kv[masked, 512 + 7] = low
    check_any_size(c.run(kernel), c.exact(), value)
    if value == "lowest" and dtype == torch.bfloat16:
        c.kv[:, 512 + 7] = low                                   # (all scores are -2.4e37 in 64 bits too)
        check_any_size(c.run(kernel), c.exact(), "all masked")


def test_a_call_of_seconds():
    """256 requests of one head over 35 million rows each (one page, over and over): 140 million tiles, some
    2.5 seconds. All scores are 0 and all rows are equal, so the output is the row, to the bit: the sums of
    powers of two are exact, and 2^-11 of a record is lost in the result's rounding to 8 bits."""
    B, page, n = 256, 65536, 35_000_000
    row = (2.0 ** torch.arange(512).remainder(7).sub(3) * (1 - 2 * torch.arange(512).remainder(2))).to(torch.bfloat16)
    kv = torch.zeros(page, 576, dtype=torch.bfloat16, device=DEV)
    kv[:, :512] = row.to(DEV)
    zeros = torch.zeros(B, 1, 576, dtype=torch.bfloat16, device=DEV)
    out = mla_prefix_decode(kv, zeros[..., :512].contiguous(), zeros[..., 512:].contiguous(), MLAConfig(0, 512, 128, 64, 1, 128),
                            group_starts=torch.tensor([0, B], dtype=torch.int32, device=DEV),
                            prefix_lens=torch.zeros(1, dtype=torch.int32, device=DEV), max_prefix_len=0,
                            seq_lens=torch.full((B,), n, dtype=torch.int32, device=DEV), max_seq_len=n, page_rows=page,
                            prefix_table=torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                            page_table=torch.zeros(B, -(-n // page), dtype=torch.int32, device=DEV), kernel=TC)
    assert torch.equal(out, row.to(DEV).expand(B, 1, 512))


@pytest.mark.parametrize("heads,batch", [(128, 512), (16, 2048)])
def test_wide_bounds_stay_on_the_tensor_cores(heads, batch):
    """Bounds of the lengths far above the lengths: the tiles that they allow (8.4 million of 128 rows at 512
    requests of 128 heads) can be counted, so the tensor-core kernel takes the call and gives the same bits as
    with bounds that fit."""
    own = [(5 * b) % 67 for b in range(batch)]
    c = Case([batch - 3, 3], [100, 33], own, heads, torch.bfloat16, 0, seed=heads)
    wide = c.run(TC, max_prefix_len=1 << 20, max_seq_len=1 << 18)
    assert torch.equal(wide, c.run(TC))
    pick = [0, 1, 13, batch // 2, batch - 4, batch - 1]
    few = Case([6], [0], [0] * 6, heads, torch.bfloat16, 0)
    few.kv, few.qa, few.qr = c.kv, c.qa[pick], c.qr[pick]
    few.sizes = [1] * 6
    few.rows_of = [c.rows_of[0] if b < batch - 3 else c.rows_of[1] for b in pick] + [c.rows_of[2 + b] for b in pick]
    check(wide[pick], few.exact(), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("own", [0, 300])
@pytest.mark.parametrize("pattern", ["stairs", "zigzag", "single", "down"])
def test_jumps_between_tiles(pattern, own, dtype):
    """Every worker has ten tiles or so of one group, and the scores of whole tiles lie 8.25 to 40 log2 units a
    step apart, up or down, each row with a step of its own (or none): the reference of a row moves past the
    rescaling threshold between any two of the sets that take the tiles in turn, for some lanes of a warp."""
    c = Case([8], [50000], [own] * 8, 16, dtype, 64, seed=41)
    g = torch.Generator().manual_seed(42)
    for r in c.rows_of:
        tiles = -(-len(r) // 64)
        t = torch.arange(tiles)
        level = {"stairs": t % 11, "zigzag": torch.randint(-6, 7, (tiles,), generator=g),
                 "single": 6 * (torch.randint(0, 4, (tiles,), generator=g) == 0), "down": 10 - t % 11}[pattern]
        c.kv[r, 512 + 9] = level.repeat_interleave(64)[:len(r)].to(dtype)
    step = torch.tensor([0.0, 8.25, -8.25, 10.0, -10.0, 16.0, -16.0, 40.0])[torch.randint(0, 8, (8, 16), generator=g)]
    c.qr[..., 9] = (step * math.log(2.0) / SCALE).to(dtype)
    check_any_size(c.run(TC), c.exact(), pattern)
