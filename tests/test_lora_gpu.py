"""linear_lora against its definition in 64 bits: token counts around the 16-token and 256-token
tiles, ragged outputs and inputs, ranks from 8 up, mixes of adapters (none, one, all different), and
values that must stay with their own request.

Tolerance. u = 2^-8 (bf16) or 2^-11 (fp16). The result's rounding is at most u of its value; A x is
rounded once, which moves the delta by at most u of sum_r |B_r (A x)_r| (here taken with absolute
values, so it is a bound and not an estimate), times the scale; fp32 sums of K products add at most
K 2^-24 of sum |w x| in the worst order, and the tensor core's accumulation is allowed twice that."""

import pytest
import torch

from latent_attn.functional import linear_lora

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(M, N, K, rank, adapters, dtype, seed=0, ids=None):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)
    if ids is None:
        ids = torch.randint(-1, adapters, (M,), generator=g, device=DEV)
    return (normal(M, K), normal(N, K, std=K ** -0.5), normal(adapters, rank, K, std=K ** -0.5),
            normal(adapters, N, rank, std=rank ** -0.5), torch.as_tensor(ids, device=DEV).to(torch.int32),
            0.25 + torch.rand(adapters, generator=g, device=DEV))


def exact(x, W, A, B, ids, scales):
    """(result, error allowed before the result's own rounding is counted) in float64."""
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -11
    x, W, A, B = x.double(), W.double(), A.double(), B.double()
    y, slack = x @ W.T, x.abs() @ W.abs().T
    slack *= 2 * x.shape[1] * 2.0 ** -24
    for a in set(ids.tolist()):
        if 0 <= a < len(A):
            at = ids == a
            s = scales[a].double() if scales is not None else 1.0
            t = s * (x[at] @ A[a].T)
            terr = u * t.abs() + abs(s) * 2 * x.shape[1] * 2.0 ** -24 * (x[at].abs() @ A[a].abs().T)
            y[at] += t @ B[a].T
            slack[at] += terr @ B[a].abs().T + 2 * A.shape[1] * 2.0 ** -24 * (t.abs() @ B[a].abs().T)
    return y, slack, u


def check(got, want):
    y, slack, u = want
    assert torch.isfinite(got).all()
    bad = (got.double() - y).abs() - (u * y.abs() + (1 + u) * slack + 2.0 ** -25)
    assert float(bad.max()) <= 0, float(bad.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 64, 255, 256, 257, 300, 600])
def test_tokens(M, dtype):
    a = make(M, 200, 320, 16, 5, dtype, seed=M)
    check(linear_lora(*a[:5], scales=a[5]), exact(*a))


@pytest.mark.parametrize("N,K", [(1, 8), (127, 64), (128, 72), (129, 4096), (443, 2504), (7168, 1024), (19000, 256),
                                 (40000, 512)])
@pytest.mark.parametrize("M", [3, 130])
def test_shapes(N, K, M):
    """Outputs that end inside a tile, odd row pitches of the result, K that ends inside a stage, one tile
    cut over many CTAs, whole rounds of tiles and a cut rest."""
    a = make(M, N, K, 24, 3, torch.bfloat16, seed=N + K)
    check(linear_lora(*a[:5], scales=a[5]), exact(*a))


@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 128, 256])
@pytest.mark.parametrize("M", [5, 200])
def test_ranks(rank, M):
    a = make(M, 384, 512, rank, 6, torch.float16, seed=rank)
    check(linear_lora(*a[:5]), exact(*a[:5], None))


@pytest.mark.parametrize("M", [7, 256, 520])
def test_mixes(M):
    n = 40
    for name, ids in (("none", [-1] * M), ("one", [3] * M), ("all different", [i % n for i in range(M)]),
                      ("runs", [i // 37 % n for i in range(M)]), ("last only", [-1] * (M - 1) + [n - 1]),
                      ("outside the loaded ones", [n + i if i % 2 else -5 for i in range(M)])):
        a = make(M, 260, 328, 16, n, torch.bfloat16, seed=M, ids=ids)
        check(linear_lora(*a[:5], scales=a[5]), exact(*a))


def test_many_adapters():
    a = make(256, 512, 256, 16, 700, torch.bfloat16, seed=1, ids=torch.randperm(700)[:256])
    check(linear_lora(*a[:5], scales=a[5]), exact(*a))


@pytest.mark.parametrize("N", [300, 20000])
def test_a_broken_adapter_stays_with_its_requests(N):
    x, W, A, B, ids, scales = make(20, N, 256, 16, 4, torch.bfloat16, ids=[i % 5 - 1 for i in range(20)])
    B[2, 7, 3], B[2, 9, 0], A[2, 1, 5] = float("nan"), float("inf"), float("inf")
    got = linear_lora(x, W, A, B, ids, scales=scales)
    hit = ids == 2
    assert not torch.isfinite(got[hit]).all(1).any()
    keep = [x[~hit], W, A, B, ids[~hit], scales]
    check(got[~hit], exact(*keep))


def test_not_finite_tokens_and_weights():
    x, W, A, B, ids, scales = make(18, 200, 256, 16, 4, torch.float16)
    x[4, 100], W[50, 3] = float("nan"), float("inf")
    got = linear_lora(x, W, A, B, ids, scales=scales)
    assert torch.isnan(got[4]).all() and not torch.isfinite(got[:, 50]).any()
    rows, cols = [i for i in range(18) if i != 4], [i for i in range(200) if i != 50]
    check(got[rows][:, cols], exact(x[rows], W[cols], A, B[:, cols], ids[rows], scales))


def test_strided_broadcast_and_given_outputs():
    x, W, A, B, ids, scales = make(33, 300, 256, 16, 4, torch.bfloat16)
    wide = torch.zeros(33, 320, dtype=torch.bfloat16, device=DEV)
    wide[:, 16:272] = x
    out = torch.empty(33, 300, dtype=torch.bfloat16, device=DEV)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    assert linear_lora(wide[:, 16:272], W, A, B, ids, scales=scales, out=out, workspace=ws) is out
    check(out, exact(x, W, A, B, ids, scales))
    same = x[:1].expand(33, 256)
    check(linear_lora(same, W, A, B, ids, scales=scales), exact(same, W, A, B, ids, scales))
    assert linear_lora(x[:0], W, A, B, ids[:0]).shape == (0, 300)


def test_same_bits_every_time():
    """Cut tiles are added in a fixed order, whichever CTA comes last; also on a side stream, with other
    work between, and in a CUDA graph."""
    a = make(67, 1000, 8192, 16, 12, torch.bfloat16, seed=3)
    first = linear_lora(*a[:5], scales=a[5])
    check(first, exact(*a))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            again = linear_lora(*a[:5], scales=a[5])
            other = make(5, 300, 512, 16, 2, torch.bfloat16)
            linear_lora(*other[:5])
            assert torch.equal(first, again)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_lora(*a[:5], scales=a[5])
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_refusals():
    x, W, A, B, ids, scales = make(4, 64, 64, 16, 2, torch.bfloat16)

    def refuses(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            linear_lora(*a, **kw)
    refuses("W must be", x, W.half(), A, B, ids)
    refuses("lora_a must be", x, W, A[:, :, :32].contiguous(), B, ids)
    refuses("lora_b must be", x, W, A, B[:1], ids)
    refuses("adapter_ids", x, W, A, B, ids.long())
    refuses("adapter_ids", x, W, A, B, ids[:3])
    refuses("scales", x, W, A, B, ids, scales=scales.half())
    refuses("out must be", x, W, A, B, ids, out=torch.empty(4, 64, device=DEV))
    refuses("2D", x[0], W, A, B, ids)
    refuses("rank", x, W, A[:, :12].contiguous(), B[..., :12].contiguous(), ids)
    refuses("multiples of 8", x[:, :60].contiguous(), W[:, :60].contiguous(), A[..., :60].contiguous(), B, ids)
    refuses("num_adapters", x, W, A[:0], B[:0], ids)
    refuses("aligned", torch.empty(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, 64), W, A, B, ids)


def test_workspaces_that_the_kernels_cannot_write_are_refused():
    x, W, A, B, ids, scales = make(40, 64, 64, 16, 2, torch.bfloat16)
    for ws in (torch.empty(64 << 20, dtype=torch.uint8), torch.empty(64 << 20, dtype=torch.uint8).pin_memory(),
               torch.empty(1, dtype=torch.uint8, device=DEV).expand(64 << 20)):
        with pytest.raises(RuntimeError, match="workspace must be"):
            linear_lora(x, W, A, B, ids, scales=scales, workspace=ws)
    check(linear_lora(x, W, A, B, ids, scales=scales, workspace=torch.empty(1, dtype=torch.uint8, device=DEV)),
          exact(x, W, A, B, ids, scales))                        # too small: one is allocated


@pytest.mark.parametrize("M", [1, 2, 3, 40, 200, 300])
def test_intermediates_beyond_the_range_of_fp16(M):
    """A x of up to some 10^6 before a small B: every output is finite, whichever tokens pass 65504."""
    x, W, A, B, ids, scales = make(M, 300, 512, 24, 5, torch.float16, seed=M)
    A = A * 512.0
    x[::3] *= 800.0
    W, B = W * 2.0 ** -4, B * 2.0 ** -13
    t = (x.double() @ A[ids.clamp(min=0)[0]].double().T).abs()
    ids[0] = 1
    assert float((x[:1].double() @ A[1].double().T).abs().max() * scales[1]) > 65504 and float(t.max()) < 1e8
    got = linear_lora(x, W, A, B, ids, scales=scales)
    check(got, exact(x, W, A, B, ids, scales))


@pytest.mark.parametrize("M,N", [(256, 25600), (200, 38000), (600, 15400), (1100, 9000), (2051, 5120)])
@pytest.mark.parametrize("mix", ["each its own", "runs", "random"])
def test_whole_rounds_then_slices(mix, M, N):
    """More tiles than CTA pairs, with one and several token blocks: pairs that go from whole tiles to a slice of
    a tile's columns, where other adapters have tokens than in the whole."""
    n = 24
    ids = None if mix == "random" else [i % n if mix == "each its own" else i // 31 % n for i in range(M)]
    a = make(M, N, 136, 24, n, torch.bfloat16, seed=M, ids=ids)
    check(linear_lora(*a[:5], scales=a[5]), exact(*a))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(67, 1000, 1000), (31, 300, 264), (256, 1030, 328), (300, 700, 96), (5, 33, 8)])
def test_every_kind_of_broken_operand(M, N, K, dtype):
    """NaN and infinities in one adapter's B (everywhere, or one row), in its A, in one token and in one row of W: an
    output is as without them where its own operands are whole, and not finite where its own sum is not."""
    n = 6
    x, W, A, B, ids, scales = make(M, N, K, 24, n, dtype, seed=M, ids=[i % (n + 1) - 1 for i in range(M)])
    want, slack, u = exact(x, W, A, B, ids, scales)

    def run(broken, x=x, W=W, A=A, B=B):
        got = linear_lora(x, W, A, B, ids, scales=scales)
        assert not torch.isfinite(got[broken]).any()
        keep = ~broken
        bad = ((got.double() - want).abs() - (u * want.abs() + (1 + u) * slack + 2.0 ** -25))[keep]
        assert torch.isfinite(got[keep]).all() and float(bad.max()) <= 0, float(bad.max())

    def hit(tokens=None, rows=None):
        m = torch.ones(M, N, dtype=torch.bool, device=DEV)
        if tokens is not None:
            m &= tokens[:, None]
        if rows is not None:
            m &= rows[None, :]
        return m
    every = torch.arange(M, device=DEV)
    for value in (float("nan"), float("inf")):
        b = B.clone()
        b[2] = value                                              # inf: of either sign by U's, but never finite
        run(hit(tokens=ids == 2), B=b)
        b = B.clone()
        b[2, N // 2, 5] = value
        run(hit(ids == 2, torch.arange(N, device=DEV) == N // 2), B=b)
        a = A.clone()
        a[1, 3, K // 2] = value
        run(hit(tokens=ids == 1), A=a)
        t = x.clone()
        t[4, K - 1] = value
        run(hit(tokens=every == 4), x=t)
        w = W.clone()
        w[N - 1, 0] = value
        run(hit(rows=torch.arange(N, device=DEV) == N - 1), W=w)


def test_a_broken_adapter_does_not_hold_up_the_batch():
    """One NaN adapter of 12 beside 67 tokens: its tokens' neighbours are computed again, in some milliseconds at
    most (element by element it was 150, the call itself 0.07)."""
    x, W, A, B, ids, scales = make(67, 7168, 16384, 16, 12, torch.bfloat16, seed=1)
    B[int(ids[ids >= 0][0])] = float("nan")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    linear_lora(x, W, A, B, ids, scales=scales)
    start.record()
    linear_lora(x, W, A, B, ids, scales=scales)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 30
