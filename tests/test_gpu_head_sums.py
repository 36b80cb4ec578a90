"""The output-head operators where long sums and small differences show,
against 64-bit results."""
import pytest

import head_cases as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def ctx(torch):
    from qwenium_b200 import qsamp

    return qsamp.Context(0)


def within(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert not off.isnan().any() and off.max() <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside, by {off.max():.3g}"


def confident_inputs(torch, N, V, D, top, cap):
    """Row n has its target's logit at `top` and one runner-up that leaves it a
    loss between 1e-6 and 1e-4; every target and runner-up is a token of its
    own, all other logits lie near 0."""
    g = torch.Generator().manual_seed(N + D)
    h = torch.randn((N, D), generator=g)
    h = H.bf16(h).double()
    unit = h / (h * h).sum(dim=1, keepdim=True)
    below = -torch.log(10.0 ** (-6 + 2 * torch.rand((N, 1), generator=g, dtype=torch.float64)))
    second = top - below
    first = torch.full_like(second, top)
    if cap:
        first, second = cap * torch.atanh(first / cap), cap * torch.atanh(second / cap)
    w = torch.randn((V, D), generator=g) * (0.3 / D**0.5)
    w[:N] = (unit * first).float()
    w[N:2 * N] = (unit * second).float()
    order = torch.randperm(V, generator=g)
    w = H.bf16(w)[torch.argsort(order)]  # token i moves to place order[i]
    t = order[:N].to(torch.int32)
    return tuple(x.cuda() for x in (H.bf16(h.float()), w, t))


@pytest.mark.parametrize("cap", [0.0, 40.0, 100.0])
@pytest.mark.parametrize("N,D", [(3, 4160), (20, 8192), (40, 4096), (64, 2048), (65, 4160), (150, 8192), (300, 4096)])
def test_gradients_of_confident_rows(torch, ctx, N, D, cap):
    """Losses of 1e-6 to 1e-4: dz of the target is minus the loss, what is left of
    exp(l - lse) - 1. The gradients make the loss's logits again, bit for bit, so
    an error common to a row's logits cancels, and what remains is:

      lse's rounding, U32 lse; the sum's (one rounding where the runner-up is
      added, its neighbours do not move a sum of 1, and the joins of few parts) and
      the exponentials beside 1: 24 U32 together;
      the runner-up's distance, off by at most both logits' errors ez (D + 8 products
      and sums; 32 U32 of the cap), times its p."""
    top = 28.0
    V = 2 * N + 300
    h, w, t = confident_inputs(torch, N, V, D, top, cap)
    g = torch.rand((N,), generator=torch.Generator().manual_seed(1)).add(0.5).cuda()
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    ez = (D + 8) * H.U32 * (hd.abs() @ wd.abs().t()).amax(dim=1)
    slope = torch.ones_like(z)
    if cap:
        y = torch.tanh(z / cap)
        z, slope = cap * y, 1 - y * y
        ez = ez + 32 * H.U32 * cap
    at = t.long()[:, None]
    lse = torch.logsumexp(z, dim=1)
    p = torch.exp(z - lse[:, None])
    rest = p.scatter(1, at, 0.0).sum(dim=1)
    assert (rest > 5e-7).all() and (rest < 2e-4).all()
    dz = p.scatter(1, at, -rest[:, None]) * slope * g.double()[:, None]
    loss, lse32 = ctx.head_loss(h, w, t, softcap=cap)
    dh, dw = ctx.head_loss_grad(h, w, t, lse32, g, softcap=cap)
    e = (lse + 24) * H.U32
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    # the target's dz, and the runner-up's (p times twice its errors); the slope is off by 2 ez / cap + 8 U32
    edz = hot * (e + 2 * ez * rest)[:, None] + (1 - hot) * p * (2 * ez + e)[:, None]
    edz = edz * slope * g.double()[:, None] + dz.abs() * (H.U16**2 if N <= 64 else H.U16)
    if cap:
        edz = edz + dz.abs() / slope * (2 * ez / cap + 8 * H.U32)[:, None]
    edz = edz + 2.0**-126
    loose = 1 + 2 * H.U16
    # d_weight of a target: its own row, and p of the others
    want = dz.t() @ hd
    bound = edz.t() @ hd.abs() * loose + (N + 64) * H.U32 * (dz.abs().t() @ hd.abs()) + H.U16 * want.abs()
    rows = t.long()
    within(dw[rows], want[rows], bound[rows], "d_weight of the targets")
    within(dw, want, bound, "d_weight")
    want = dz @ wd
    bound = edz @ wd.abs() * loose + (V + 64) * H.U32 * (dz.abs() @ wd.abs()) + H.U16 * want.abs()
    within(dh, want, bound, "d_hidden")
    # and the loss itself: lse's rounding, the target's logit is the largest
    within(loss, lse - z.gather(1, at)[:, 0], e + 2 * ez * rest, "loss")


@pytest.mark.parametrize("N,D", [(50, 64), (150, 64), (50, 4096), (150, 4096)])
def test_gradients_of_large_logits(torch, ctx, N, D):
    """Logits of a few thousand, rows whose largest is 60 above the next: lse is
    that logit to the bit (logf(1) is 0), p is 1 there and 0 elsewhere, so dz is g
    at the largest, -g at the target, and at most 8 U32 g where they meet."""
    V = 2000
    h, w, t, g = H.head_inputs(N, V, D, seed=6, scale=2000.0, ignored=0.0, device="cuda")
    hd, wd = h.double(), w.double()
    top2, arg = (hd @ wd.t()).topk(2, dim=1)
    clear = top2[:, 0] - top2[:, 1] > 60
    assert clear.sum() > N // 2
    t = torch.where(torch.arange(N, device="cuda") % 3 == 0, arg[:, 0].to(torch.int32), t)  # some are their targets
    t = torch.where(clear, t, -1)
    _, lse = ctx.head_loss(h, w, t)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    gr = torch.where(t >= 0, g, 0.0).double()[:, None]
    hot = torch.zeros((N, V), dtype=torch.float64, device="cuda").scatter_(1, t.long().clamp(min=0)[:, None], 1.0)
    p = torch.zeros_like(hot).scatter_(1, arg[:, :1], 1.0)
    dz = (p - hot) * gr
    edz = dz.abs() * (H.U16**2 if N <= 64 else H.U16) + 8 * H.U32 * (p + hot) * gr.abs() + 2.0**-80
    loose = 1 + 2 * H.U16
    want = dz @ wd
    within(dh, want, edz @ wd.abs() * loose + (V + 64) * H.U32 * (dz.abs() @ wd.abs()) + H.U16 * want.abs(), "d_hidden")
    want = dz.t() @ hd
    within(dw, want, edz.t() @ hd.abs() * loose + (N + 64) * H.U32 * (dz.abs().t() @ hd.abs()) + H.U16 * want.abs(), "d_weight")


@pytest.mark.parametrize("more", [1, 40, 64])
def test_a_last_round_of_few_rows(torch, ctx, more):
    """Rows past a round of partial sums: a row's bits are those it has in the
    first round, however few rows the last one holds."""
    D, V = 2048, 200
    h, w, t, _ = H.head_inputs(16384, V, D, seed=18, device="cuda")
    h, t = torch.cat([h, h[:more]]), torch.cat([t, t[:more]])
    loss, lse = ctx.head_loss(h, w, t)
    assert torch.equal(lse[16384:], lse[:more]) and torch.equal(loss[16384:], loss[:more])


def test_a_long_sum_of_one_sign(torch, ctx):
    """d_weight over 2^22 rows whose terms have one sign: logits 0, so dz is -7/8
    and 1/8 to the bit. In tensor memory an addition cuts 16 products and the sum
    so far, each by at most 2^-23 of that sum: over a slice of 2048 additions, the
    sum half its last on average, 17 * 2^-13 of it; the slices' sum adds 128 U32;
    one rounding to bf16. (2^21 rows in one slice came out low by 1.2e-2.)"""
    N, V, D = 2**22, 8, 64
    gen = torch.Generator(device="cuda").manual_seed(19)
    h = (torch.rand((N, D), generator=gen, device="cuda") * 0.5 + 0.5).to(torch.bfloat16)
    w = torch.zeros((V, D), dtype=torch.bfloat16, device="cuda")
    t = torch.zeros((N,), dtype=torch.int32, device="cuda")
    _, lse = ctx.head_loss(h, w, t)
    _, dw = ctx.head_loss_grad(h, w, t, lse, torch.ones((N,), device="cuda"))
    total = h.double().sum(dim=0)
    # exp(-lse) is within 8 U32 of 1/8, and so rounds to it
    want = torch.cat([-0.875 * total[None], 0.125 * total[None].expand(V - 1, D)])
    bound = (H.U16 + (17 * 2.0**-13 + 128 * H.U32) * (1 + H.U16)) * want.abs()
    within(dw, want, bound, "d_weight")


def test_long_sums_over_the_vocabulary(torch, ctx):
    """d_hidden in two pieces of the vocabulary whose sums are several slices each
    (many tiles of d_hidden leave no room for splits), d_weight beside it in one;
    the last piece's rows, one of them a target, among d_weight's."""
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GB")
    N, V, D = 1100, 200000, 8200
    gen = torch.Generator(device="cuda").manual_seed(21)
    w = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    for r in range(0, V, 20000):
        w[r:r + 20000] = torch.randn((20000, D), generator=gen, device="cuda") * (2.0 / D**0.5)
    h = torch.randn((N, D), generator=gen, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, V, (N,), generator=gen, device="cuda").to(torch.int32)
    t[0], t[5] = V - 1, -1
    g = torch.rand((N,), generator=gen, device="cuda") + 0.5
    z = torch.cat([h.double() @ w[r:r + 20000].double().t() for r in range(0, V, 20000)], dim=1)
    lse64 = torch.logsumexp(z, dim=1)
    _, lse = ctx.head_loss(h, w, t)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    dz = torch.exp(z - lse64[:, None])
    dz.scatter_add_(1, t.long().clamp(min=0)[:, None], torch.full((N, 1), -1.0, dtype=torch.float64, device="cuda"))
    dz *= torch.where(t >= 0, g, 0.0).double()[:, None]
    want = sum(dz[:, r:r + 20000] @ w[r:r + 20000].double() for r in range(0, V, 20000))
    # two independent roundings of half a bf16 step each stay below twice one of them
    assert (dh.double() - want).norm() <= 2 * H.U16 * want.norm() and (dh[5] == 0).all()
    for a in (0, 100000 - 1000, V - 2000):
        want = dz[:, a:a + 2000].t() @ h.double()
        assert (dw[a:a + 2000].double() - want).norm() <= 2 * H.U16 * want.norm()


def rounded_e4m3(torch, y):
    """Doubles to the nearest e4m3 value, ties to even, saturated."""
    y = y.clamp(-448.0, 448.0)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs())[1].sub(1).clamp(min=-6).sub(3))
    return torch.round(y / step) * step


@pytest.mark.parametrize("rows,M", [(1, 65535 * 32 + 33), (128, 65535 * 128 + 129)])
def test_quantiser_rows_past_the_grid(torch, ctx, rows, M):
    """More groups of rows (32, or a square block) than a grid's second dimension
    holds: its blocks take a second group. Every group has its own scale."""
    K = 16
    if torch.cuda.mem_get_info()[0] < 20 * 2**30:
        pytest.skip("needs 20 GB")
    r = torch.arange(M, device="cuda")
    x = torch.rand((M, K), generator=torch.Generator(device="cuda").manual_seed(20), device="cuda") - 0.5
    x *= torch.ldexp(1 + (r // rows % 127).float() / 128, (r // rows % 41 - 20).to(torch.int32))[:, None]
    x = x.to(torch.bfloat16)
    q, s = ctx.quantize_fp8(x, block_rows=rows)
    blocks = -(-M // rows)
    top = torch.zeros((blocks * rows,), dtype=torch.float64, device="cuda")
    top[:M] = x.abs().amax(dim=1).double()
    top = top.view(blocks, rows).amax(dim=1, keepdim=True)
    assert torch.equal(s, (top / torch.full_like(top, 448.0)).float())
    for a in range(0, M, 2**20):
        b = min(a + 2**20, M)
        want = rounded_e4m3(torch, x[a:b].double() / s[r[a:b] // rows].double())
        assert torch.equal(q[a:b].double(), want), f"rows {a} to {b}"
