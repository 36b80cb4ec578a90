"""The output-head operators against 64-bit results: cross entropy over a head
without kept logits and its gradients, the 8-bit block-scaled product, the
quantiser; strides, empty and odd sizes, masks, streams, captured graphs, and
a run of them with the selection that reads the head's logits."""
import numpy as np
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
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, what
    nan = want.isnan()
    assert (got.isnan() == nan).all(), f"{what}: NaN where none belongs, or none where one does"
    off = ((got - want).abs() - bound)[~nan]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside, by {off.max():.3g}"


def guarded(torch, rows, cols, pad, dtype):
    """A [rows][cols] view of stride cols + pad in a filled buffer."""
    buf = torch.full((rows + 2, cols + pad), 77.0, dtype=dtype, device="cuda")
    return buf, buf[:rows, :cols]


SIZES = [
    (1, 1, 8), (1, 2, 16), (1, 257, 64), (3, 31, 8), (5, 1000, 72), (33, 128, 40), (64, 255, 1024), (127, 256, 64),
    (130, 513, 128), (257, 4099, 264), (300, 1025, 200), (512, 300, 520), (17, 20011, 96), (700, 70, 48),
    (16, 400, 64), (32, 400, 64), (65, 400, 64), (129, 20011, 64),
]


@pytest.mark.parametrize("cap", [0.0, 30.0, 2.0, 1e5])
@pytest.mark.parametrize("N,V,D", SIZES)
def test_loss_and_gradients(torch, ctx, N, V, D, cap):
    h, w, t, g = H.head_inputs(N, V, D, seed=1, device="cuda")
    want = H.head_exact(h, w, t, g, cap, dz_error=H.U16**2 if N <= 64 else H.U16)
    loss, lse = ctx.head_loss(h, w, t, softcap=cap)
    within(loss, want["loss"], want["eloss"], "loss")
    within(lse, want["lse"], want["else"], "lse")
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g, softcap=cap)
    within(dh, want["dh"], want["edh"], "d_hidden")
    within(dw, want["dw"], want["edw"], "d_weight")
    torch.cuda.synchronize()
    ctx.poll_status()


# (4200, 70001): three pieces of the vocabulary; (30, 4300000): two, few rows; D 4160: several slices of a sum
@pytest.mark.parametrize("N,V,D", [(9, 140000, 64), (2100, 9000, 128), (40, 33000, 1536), (4200, 70001, 64),
                                   (30, 4300000, 8), (20, 2100, 4160), (300, 2100, 4160)])
def test_many_pieces_and_tiles(torch, ctx, N, V, D):
    if N * V > 10**8 and torch.cuda.mem_get_info()[0] < 60 * 2**30:
        pytest.skip("the 64-bit results need 60 GB")
    h, w, t, g = H.head_inputs(N, V, D, seed=2, device="cuda")
    want = H.head_exact(h, w, t, g, 0.0)
    loss, lse = ctx.head_loss(h, w, t)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    for got, name, e in ((loss, "loss", "eloss"), (lse, "lse", "else"), (dh, "dh", "edh"), (dw, "dw", "edw")):
        within(got, want[name], want[e], name)
    # the bounds above add every rounding up; independent ones of half a bf16 step each stay far below
    assert (dh.double() - want["dh"]).norm() <= 2 * H.U16 * want["dh"].norm()
    assert (dw.double() - want["dw"]).norm() <= 2 * H.U16 * want["dw"].norm()


def test_loss_of_many_rows(torch, ctx):
    """More rows than one round of partial sums holds."""
    h, w, t, _ = H.head_inputs(40000, 300, 64, seed=16, device="cuda")
    want = H.head_exact(h, w, t, torch.ones(40000, device="cuda"), 0.0)
    loss, lse = ctx.head_loss(h, w, t)
    within(loss, want["loss"], want["eloss"], "loss")
    within(lse, want["lse"], want["else"], "lse")


def test_gradient_against_differences(torch, ctx):
    """sum_n g[n] loss[n] moved along single coordinates: steps that bf16
    holds exactly, loss errors over the step's width, third derivative <= 8 |x|^3."""
    N, V, D, eps = 6, 700, 64, 2.0**-6
    h, w, t, g = H.head_inputs(N, V, D, seed=3, ignored=0.0, device="cuda")
    h = torch.round(h.float() * 16).clamp(-24, 24).div(16).to(torch.bfloat16)  # |h| < 2 in steps of 2^-4
    w = torch.round(w.float() * 16).clamp(-24, 24).div(16).to(torch.bfloat16)
    want = H.head_exact(h, w, t, g, 0.0)
    lse = ctx.head_loss(h, w, t)[1]
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)

    def total(hh, ww):
        return float((ctx.head_loss(hh, ww, t)[0].double() * g.double()).sum())

    err = float((want["eloss"] * g.double().abs()).sum()) / eps + eps**2 * 8 / 6 * float(g.abs().sum()) * 1.5**3
    for n, d in ((0, 0), (3, 17), (5, 63)):
        up, dn = h.clone(), h.clone()
        up[n, d] += eps
        dn[n, d] -= eps
        assert float(up[n, d]) - float(dn[n, d]) == 2 * eps
        diff = (total(up, w) - total(dn, w)) / (2 * eps)
        assert abs(diff - float(dh[n, d])) <= err + float(want["edh"][n, d])
    for v, d in ((int(t[0]), 5), (int(t[4]), 40), (123, 9)):
        up, dn = w.clone(), w.clone()
        up[v, d] += eps
        dn[v, d] -= eps
        assert float(up[v, d]) - float(dn[v, d]) == 2 * eps
        diff = (total(h, up) - total(h, dn)) / (2 * eps)
        assert abs(diff - float(dw[v, d])) <= err + float(want["edw"][v, d])


@pytest.mark.parametrize("N,dead", [(40, 1), (300, 1), (900, 600)])
def test_gradients_of_a_mean(torch, ctx, N, dead):
    """One grad_loss for all rows, in the middle between two bf16 numbers (so
    that its own rounding would be off by 2^-8 in every row alike): the
    targets' terms, all but the whole of the gradients here, keep their digits.

    The targets' dz over grad_loss is -(1 - p), whose nearest bf16 number is
    -1 for p <= 2^-9: off by p. The other terms are p, off by U16 p."""
    V, D = 2000, 64
    h, w, t, _ = H.head_inputs(N, V, D, seed=17, scale=0.01, device="cuda")
    t[:dead] = -1  # rows without a gradient, whose grad_loss is not read
    t[dead // 2 + 1:dead] = 5  # rows whose gradient is 0
    g = torch.full((N,), 1.0 + 2.0**-8, device="cuda")
    g[:dead] = float("nan")
    g[dead // 2 + 1:dead] = 0.0
    want = H.head_exact(h, w, t, g, 0.0)
    _, lse = ctx.head_loss(h, w, t)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    g = torch.where(t >= 0, g, 0.0)
    p = torch.exp(h.double() @ w.double().t() - want["lse"].unsqueeze(1))
    assert p.max() < 2.0**-9
    live = (t >= 0).unsqueeze(1)
    hot = torch.zeros_like(p).scatter_(1, t.long().clamp(min=0).unsqueeze(1), 1.0)
    # 2^-15: the exponentials and sums of p in 32 bits, relative (p itself is below 2^-9)
    edz = torch.where(live, g.double().unsqueeze(1) * (hot * p + (1 - hot) * p * (H.U16 + 2.0**-15) + 2.0**-9 * 2.0**-15), 0.0)
    dz = torch.where(live, g.double().unsqueeze(1) * (p + hot), 0.0)
    edh = (1 + H.U16) * edz @ w.double().abs() + (V + 64) * H.U32 * (dz @ w.double().abs()) + H.U16 * want["dh"].abs()
    edw = (1 + H.U16) * edz.t() @ h.double().abs() + (N + 64) * H.U32 * (dz.t() @ h.double().abs()) + H.U16 * want["dw"].abs()
    within(dh, want["dh"], edh, "d_hidden")
    within(dw, want["dw"], edw, "d_weight")


def test_rows_without_a_loss(torch, ctx):
    """Every row masked: zero losses and gradients, whatever grad_loss and lse hold."""
    h, w, t, g = H.head_inputs(70, 300, 64, seed=4, device="cuda")
    t = torch.full_like(t, -1)
    loss, lse = ctx.head_loss(h, w, t)
    assert (loss == 0).all() and torch.isfinite(lse).all()
    bad = torch.full_like(lse, float("nan"))
    dh, dw = ctx.head_loss_grad(h, w, t, bad, bad)
    assert (dh == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("N", [20, 150])
def test_whatever_lies_in_masked_rows(torch, ctx, N):
    """NaN and infinities in hidden rows without a gradient (padding behind a
    batch's sequences) reach no other row and not the weight's gradient."""
    h, w, t, g = H.head_inputs(N, 700, 64, seed=15, ignored=0.4, device="cuda")
    t[5] = 700  # past the vocabulary: no gradient either
    dead = (t < 0) | (t >= 700)
    want = H.head_exact(torch.where(dead[:, None], 0.0, h), w, t, g, 0.0)
    bad = h.clone()
    bad[dead] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").repeat(16).to(torch.bfloat16)
    loss, lse = ctx.head_loss(bad, w, t)
    keep = t >= 700
    assert (loss[dead & ~keep] == 0).all()
    within(loss[~dead], want["loss"][~dead], want["eloss"][~dead], "loss")
    dh, dw = ctx.head_loss_grad(bad, w, t, lse, torch.where(dead, float("nan"), g))
    assert (dh[dead] == 0).all()
    within(dh, want["dh"], want["edh"], "d_hidden")
    within(dw, want["dw"], want["edw"], "d_weight")


def test_no_rows(torch, ctx):
    _, w, _, _ = H.head_inputs(1, 300, 64, device="cuda")
    h = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    e = torch.empty((0,), dtype=torch.float32, device="cuda")
    t = torch.empty((0,), dtype=torch.int32, device="cuda")
    loss, lse = ctx.head_loss(h, w, t)
    assert loss.shape == (0,) and lse.shape == (0,)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, e)
    assert dh.shape == (0, 64) and (dw == 0).all() and dw.shape == w.shape


def test_target_past_the_vocabulary(torch, ctx):
    """NaN loss, no gradient; the other rows keep theirs."""
    h, w, t, g = H.head_inputs(40, 500, 64, seed=5, device="cuda")
    t[7], t[9] = 500, 2**31 - 1
    want = H.head_exact(h, w, t, g, 0.0)
    loss, lse = ctx.head_loss(h, w, t)
    within(loss, want["loss"], want["eloss"], "loss")
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    assert (dh[7] == 0).all() and (dh[9] == 0).all()
    within(dh, want["dh"], want["edh"], "dh")
    within(dw, want["dw"], want["edw"], "dw")


def test_large_logits(torch, ctx):
    """Logits of a few thousand: one token takes the whole row, and the sums neither overflow nor vanish."""
    h, w, t, g = H.head_inputs(50, 2000, 64, seed=6, scale=2000.0, device="cuda")
    want = H.head_exact(h, w, t, g, 0.0)
    loss, lse = ctx.head_loss(h, w, t)
    within(loss, want["loss"], want["eloss"], "loss")
    within(lse, want["lse"], want["else"], "lse")
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    # p of a runner-up moves by its logit's error, up to 1 for these logits: edh already counts that (p e)
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


def test_a_bad_row_stays_alone(torch, ctx):
    """A NaN in one hidden row: that row's results are NaN, the others' are not touched."""
    h, w, t, g = H.head_inputs(40, 500, 64, seed=7, ignored=0.0, device="cuda")
    loss0, lse0 = ctx.head_loss(h, w, t)
    dh0, _ = ctx.head_loss_grad(h, w, t, lse0, g)
    h2 = h.clone()
    h2[11, 3] = float("nan")
    loss, lse = ctx.head_loss(h2, w, t)
    dh, _ = ctx.head_loss_grad(h2, w, t, lse, g)
    ok = torch.arange(40, device="cuda") != 11
    assert loss[11].isnan() and lse[11].isnan() and dh[11].isnan().all()
    assert torch.equal(loss[ok], loss0[ok]) and torch.equal(lse[ok], lse0[ok]) and torch.equal(dh[ok], dh0[ok])


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("N", [20, 150])
def test_logits_of_minus_infinity(torch, ctx, N, cap):
    """Finite factors whose product passes fp32's range, as the first and the
    last token's logit of each row: without a soft-cap these tokens take no part
    and have no gradient, as though they were not there; with one their logit is -cap."""
    V, D = 400, 64
    h, w, t, g = H.head_inputs(N, V, D, seed=16, device="cuda")
    h[:, 0] = 4.0
    w[:, 0] = 0.0
    low = torch.zeros((1, D), dtype=torch.bfloat16, device="cuda")
    low[0, 0] = -(2.0**127)
    wide = torch.cat([low, w, low])
    at = torch.where(t >= 0, t + 1, t)
    loss, lse = ctx.head_loss(h, wide, at, softcap=cap)
    dh, dw = ctx.head_loss_grad(h, wide, at, lse, g, softcap=cap)
    assert torch.isfinite(loss).all() and torch.isfinite(lse).all()
    # dz of the two tokens is exactly 0: exp(-inf), or a slope 1 - (l / cap)^2 of at most a rounding, times -2^127
    assert torch.isfinite(dh[:, 1:]).all() and torch.isfinite(dw[1:-1]).all()
    if cap == 0.0:
        assert (dw[0] == 0).all() and (dw[-1] == 0).all()
        want = H.head_exact(h, w, t, g, 0.0)
        within(loss, want["loss"], want["eloss"], "loss")
        within(lse, want["lse"], want["else"], "lse")
        within(dh, want["dh"], want["edh"], "d_hidden")
        within(dw[1:-1], want["dw"], want["edw"], "d_weight")


def test_strided_matrices_and_guards(torch, ctx):
    """Views with their own strides give the same bits; nothing outside the outputs is written."""
    N, V, D = 131, 777, 72
    h, w, t, g = H.head_inputs(N, V, D, seed=8, device="cuda")
    loss, lse = ctx.head_loss(h, w, t)
    dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
    bh, vh = guarded(torch, N, D, 24, torch.bfloat16)
    bw, vw = guarded(torch, V, D, 8, torch.bfloat16)
    vh.copy_(h)
    vw.copy_(w)
    bdh, vdh = guarded(torch, N, D, 40, torch.bfloat16)
    bdw, vdw = guarded(torch, V, D, 16, torch.bfloat16)
    loss2, lse2 = ctx.head_loss(vh, vw, t)
    ctx.head_loss_grad(vh, vw, t, lse2, g, d_hidden=vdh, d_weight=vdw)
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2) and torch.equal(dh, vdh) and torch.equal(dw, vdw)
    for buf, rows, cols in ((bdh, N, D), (bdw, V, D), (bh, N, D), (bw, V, D)):
        assert (buf[rows:] == 77).all() and (buf[:, cols:] == 77).all()


def test_same_bits_every_time(torch, ctx):
    h, w, t, g = H.head_inputs(600, 5000, 256, seed=9, device="cuda")
    first = None
    for _ in range(4):
        loss, lse = ctx.head_loss(h, w, t)
        dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
        if first is None:
            first = (loss, lse, dh, dw)
        else:
            assert all(torch.equal(a, b) for a, b in zip(first, (loss, lse, dh, dw)))


# ---------------------------------------------------------------- quantiser
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K,pad", [(1, 1, 0), (3, 127, 0), (2, 128, 0), (5, 300, 3), (130, 257, 1), (129, 512, 8), (7, 1000, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantiser(torch, ctx, M, K, pad, rows, dtype):
    g = torch.Generator().manual_seed(M * K + rows)
    x = torch.randn((M, K), generator=g) * torch.exp(3 * torch.randn((M, 1), generator=g))
    if M > 2:
        x[1] = 0
    x = x.to(getattr(torch, dtype))
    buf = torch.zeros((M, K + pad), dtype=x.dtype, device="cuda")
    view = buf[:, :K]
    view.copy_(x)
    q, s = ctx.quantize_fp8(view, block_rows=rows)
    wq, ws = H.quant_exact(x, rows)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu().double(), wq)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantiser_borders(torch, ctx, dtype):
    """Values on and beside the borders between two e4m3 values, subnormal
    codes, tiny and huge blocks, infinities and NaN."""
    grid = torch.arange(127, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (grid[1:] + grid[:-1]) / 2
    rows = []
    for scale in (1.0, 0.37, 3e-30, 1e-38, 1e30, 7e35):
        v = torch.zeros(256)
        v[0] = 448.0
        v[1:127] = mid
        v[128] = -448.0
        v[129:256] = -torch.cat([mid, mid[-1:]]) * (1 + 2.0**-20)
        rows.append(v * scale)
    x = torch.stack(rows)
    bad = torch.ones((3, 256))
    bad[0, 5], bad[1, 200], bad[2, 0] = float("inf"), float("nan"), float("-inf")
    x = torch.cat([x, bad]).to(getattr(torch, dtype))
    q, s = ctx.quantize_fp8(x.cuda())
    wq, ws = H.quant_exact(x, 1)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(ws, nan=-1.0))
    assert torch.equal(torch.nan_to_num(q.cpu().double(), nan=-1.0), torch.nan_to_num(wq, nan=-1.0))


def rounded_e4m3(torch, y):
    """Doubles to the nearest e4m3 value, ties to even, saturated."""
    y = y.clamp(-448.0, 448.0)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs())[1].sub(1).clamp(min=-6).sub(3))
    return torch.round(y / step) * step


def test_quantiser_every_bf16(torch, ctx):
    """Every bf16 magnitude below a block's largest, for many largest ones:
    the codes of the exact quotients. (The quotient of a bf16 by a 32-bit scale
    is never within 2^-53 of a border without lying on it.)"""
    allv = torch.arange(1, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    tops = [1.0, 1.5, 448.0, 7.0, 3.5, 1.9921875, 2.0**-60, 2.0**-120, 2.0**100]
    tops += (1 + torch.randint(0, 128, (24,), generator=g) / 128).tolist()
    for top in tops:
        v = allv[(allv.float() <= top) & (allv.float() >= top * 2.0**-22)]
        v = torch.cat([v, -v])
        n = -(-v.numel() // 127)
        x = torch.zeros((n * 127,), dtype=torch.bfloat16)
        x[:v.numel()] = v
        x = torch.cat([torch.full((n, 1), top, dtype=torch.bfloat16), x.reshape(n, 127)], dim=1).cuda()
        q, s = ctx.quantize_fp8(x)
        assert (s == torch.tensor(top, dtype=torch.float64).div(448).float().item()).all()
        want = rounded_e4m3(torch, x.double() / s.double())
        assert torch.equal(q.double(), want), f"largest {top}: {int((q.double() != want).sum())} codes differ"


@pytest.mark.parametrize("exponent", [0, 40, -45, 127])
def test_scale_of_every_mantissa(torch, ctx, exponent):
    """The scale is the largest value over 448, rounded once."""
    bits = torch.arange(2**23, dtype=torch.int32, device="cuda") | ((exponent + 127) << 23)
    x = bits.view(torch.float32).reshape(-1, 1)
    q, s = ctx.quantize_fp8(x)
    want = x.double() / torch.full_like(x, 448.0, dtype=torch.float64)  # 53 bits: 24 of them over 7 need no second look
    assert torch.equal(s, want.float())
    assert (q.float() == 448).all()


@pytest.mark.parametrize("rows", [1, 128])
def test_quantiser_large(torch, ctx, rows):
    """Random values over many binades in blocks of both shapes, both types."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((1000, 2000), generator=g, device="cuda")
    x *= torch.exp(4 * torch.randn((1000, 1), generator=g, device="cuda"))
    for t in (torch.float32, torch.bfloat16):
        v = x.to(t)
        q, s = ctx.quantize_fp8(v, block_rows=rows)
        blocks = torch.nn.functional.max_pool2d(v.double().abs()[None], (rows, 128), ceil_mode=True)[0]
        assert torch.equal(s, (blocks / torch.full_like(blocks, 448.0)).float())
        spread = s.double().repeat_interleave(rows, 0)[:1000].repeat_interleave(128, 1)[:, :2000]
        assert torch.equal(q.double(), rounded_e4m3(torch, v.double() / spread))


def test_quantiser_many_rows(torch, ctx):
    """More rows than a grid's second dimension holds."""
    x = torch.full((70000, 16), 2.0, dtype=torch.bfloat16, device="cuda")
    q, s = ctx.quantize_fp8(x)
    assert (q.float() == 448).all() and (s == torch.tensor(2.0) / 448).all()


# ---------------------------------------------------------------- 8-bit product
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("M,V,K", [(1, 1, 1), (1, 129, 128), (2, 300, 16), (10, 1001, 400), (33, 255, 127), (128, 128, 256),
                                   (129, 4097, 513), (256, 512, 1024), (300, 700, 1000), (1000, 130, 2056),
                                   (16, 300, 260), (17, 300, 260), (64, 300, 260), (65, 300, 260), (20, 30011, 300),
                                   (600, 20011, 2100), (100, 300, 8320), (5, 200, 66000)])
def test_product(torch, ctx, M, V, K, f32):
    x, sx, w, sw = H.fp8_inputs(M, V, K, device="cuda")
    kp = -(-K // 16) * 16
    xp = torch.zeros((M, kp), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :K]
    wp = torch.full((V, kp + 16), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :K]
    xp.copy_(x)
    wp.copy_(w)
    want, bound = H.fp8_exact(x, sx, w, sw)
    dtype = torch.float32 if f32 else torch.bfloat16
    out = ctx.matmul_fp8(xp, sx, wp, sw, out_dtype=dtype)
    within(out, want, bound if f32 else bound + H.U16 * want.abs() + bound * H.U16 + 2.0**-126, "product")
    # every alignment of the output, guarded
    for pad in (1, 3):
        buf = torch.full((M + 1, V + pad), 77.0, dtype=dtype, device="cuda")
        view = buf[:M, pad:]
        ctx.matmul_fp8(xp, sx, wp, sw, out=view)
        assert torch.equal(view, out)
        assert (buf[M] == 77).all() and (buf[:, :pad] == 77).all()


def test_product_nan_block(torch, ctx):
    """A block with a NaN scale makes its row (activations) or its 128 columns (weights) NaN, nothing else."""
    x, sx, w, sw = H.fp8_inputs(20, 400, 256, seed=2, device="cuda")
    out0 = ctx.matmul_fp8(x, sx, w, sw)
    sx2, sw2 = sx.clone(), sw.clone()
    sx2[3, 1] = float("nan")
    sw2[2, 0] = float("nan")
    out = ctx.matmul_fp8(x, sx2, w, sw2)
    bad = torch.zeros((20, 400), dtype=torch.bool, device="cuda")
    bad[3] = True
    bad[:, 256:384] = True
    assert out[bad].isnan().all() and torch.equal(out[~bad], out0[~bad])


def test_product_strided_scales(torch, ctx):
    x, sx, w, sw = H.fp8_inputs(50, 300, 384, seed=3, device="cuda")
    out = ctx.matmul_fp8(x, sx, w, sw)
    bx = torch.full((50, 8), float("nan"), device="cuda")
    bw = torch.full((3, 5), float("nan"), device="cuda")
    bx[:, 1:4], bw[:, 2:5] = sx, sw
    assert torch.equal(out, ctx.matmul_fp8(x, bx[:, 1:4], w, bw[:, 2:5]))


# ---------------------------------------------------------------- far offsets
def roomy(torch, gib):
    if torch.cuda.mem_get_info()[0] < gib * 2**30:
        pytest.skip(f"needs {gib} GB")


def test_offsets_past_32_bits_product(torch, ctx):
    """A result of more than 2^31 elements: its last rows are those of a small call."""
    roomy(torch, 30)
    M, V, K = 8300, 262144, 128
    x, sx, w, sw = H.fp8_inputs(300, V, K, seed=5, device="cuda")
    big = torch.zeros((M, K), dtype=torch.uint8, device="cuda").view(x.dtype)
    bs = torch.zeros((M, 1), device="cuda")
    big[-300:] = x
    bs[-300:] = sx
    out = ctx.matmul_fp8(big, bs, w, sw)
    assert out.numel() > 2**31
    assert torch.equal(out[-300:], ctx.matmul_fp8(x, sx, w, sw)) and (out[:256] == 0).all()


def test_offsets_past_32_bits_quantiser(torch, ctx):
    roomy(torch, 30)
    M, K = 263000, 8192
    x = torch.randn((M, 64), device="cuda").to(torch.bfloat16).repeat(1, K // 64)
    assert x.numel() > 2**31
    for rows in (1, 128):
        q, s = ctx.quantize_fp8(x, block_rows=rows)
        tail = M // 128 * 128 - 256
        q2, s2 = ctx.quantize_fp8(x[tail:], block_rows=rows)
        assert torch.equal(q[tail:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[tail // rows:], s2)
        del q, s


def test_offsets_past_32_bits_gradients(torch, ctx):
    """A weight of more than 2^31 elements: loss and the gradients of its last
    rows (one of them a target), and of the hidden rows."""
    roomy(torch, 60)
    N, V, D = 3, 262200, 8200
    g = torch.Generator(device="cuda").manual_seed(6)
    w = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    for r in range(0, V, 30000):
        w[r:r + 30000] = torch.randn((min(30000, V - r), D), generator=g, device="cuda") * (2.0 / D**0.5)
    h = torch.randn((N, D), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.tensor([V - 1, 5, V - 200], dtype=torch.int32, device="cuda")
    z = torch.cat([h.double() @ w[r:r + 30000].double().t() for r in range(0, V, 30000)], dim=1)
    lse64 = torch.logsumexp(z, dim=1)
    loss, lse = ctx.head_loss(h, w, t)
    err = (D + 8) * H.U32 * (h.double().abs() @ w[-1000:].double().abs().t()).max() * 2 + (V + 256) * H.U32
    assert (lse - lse64).abs().max() <= err + 4 * H.U32 * lse64.max()
    assert (loss - (lse64 - z.gather(1, t.long()[:, None])[:, 0])).abs().max() <= 2 * err + 8 * H.U32 * lse64.max()
    grad = torch.tensor([1.0, -0.5, 0.25], device="cuda")
    dh, dw = ctx.head_loss_grad(h, w, t, lse, grad)
    p = torch.exp(z - lse64[:, None])
    p[torch.arange(N), t.long()] -= 1
    dz = p * grad.double()[:, None]
    want = dz[:, -300:].t() @ h.double()
    assert (dw[-300:].double() - want).norm() <= 1.01 * H.U16 * want.norm()
    want = sum(dz[:, r:r + 30000] @ w[r:r + 30000].double() for r in range(0, V, 30000))
    assert (dh.double() - want).norm() <= 1.01 * H.U16 * want.norm()


# ---------------------------------------------------------------- together
def test_serving_step(torch, ctx):
    """Quantise the hidden rows, make the head's logits in 8 bits, sample from
    them where they lie, and score the sampled tokens: the sampler's
    probability is that of the logits it read."""
    from qwenium_b200 import qsamp
    from qwenium_b200 import workloads as W

    B, D, V = 10, 512, 15001
    h, w, _, _ = H.head_inputs(B, V, D, seed=11, device="cuda")
    wq, ws = ctx.quantize_fp8(w, block_rows=128)
    hq, hs = ctx.quantize_fp8(h)
    logits = ctx.matmul_fp8(hq, hs, wq, ws, out_dtype=torch.float32)
    want, bound = H.fp8_exact(hq, hs, wq, ws)
    within(logits, want, bound, "logits")
    ids = torch.empty(B, dtype=torch.int32, device="cuda")
    p = W.default_params(B)
    res = ctx.sample_batch(logits, p, u=np.linspace(0.05, 0.95, B), out_ids=ids)
    torch.cuda.synchronize()
    ctx.poll_status()
    got = res.cpu().numpy().view(qsamp.ROW_RESULT).reshape(-1)
    lp = torch.log_softmax(want, dim=1).gather(1, ids.long().unsqueeze(1)).squeeze(1).cpu().numpy()
    # the sampler's sums are sequential fp32 over the row
    np.testing.assert_allclose(np.log(got["prob"]), lp, atol=2 * float(bound.max()) + V * H.U32)
    # the unquantised head's log-probability of the same tokens
    loss, lse = ctx.head_loss(h, w, ids)
    exact = H.head_exact(h, w, ids, torch.ones(B, device="cuda"), 0.0)
    within(loss, exact["loss"], exact["eloss"], "score")


def test_scores_match_the_sampler(torch, ctx):
    """exp(-loss) of a sampled token is the sampler's probability for the same logits."""
    from qwenium_b200 import qsamp
    from qwenium_b200 import workloads as W

    B, D, V = 12, 64, 5000
    h, w, _, _ = H.head_inputs(B, V, D, seed=12, device="cuda")
    logits = (h.double() @ w.double().t()).float()
    ids = torch.empty(B, dtype=torch.int32, device="cuda")
    res = ctx.sample_batch(logits, W.default_params(B), u=np.linspace(0.01, 0.99, B), out_ids=ids)
    torch.cuda.synchronize()
    got = res.cpu().numpy().view(qsamp.ROW_RESULT).reshape(-1)
    loss, _ = ctx.head_loss(h, w, ids)
    tol = float(H.head_exact(h, w, ids, torch.ones(B, device="cuda"), 0.0)["eloss"].max()) + V * H.U32
    np.testing.assert_allclose(np.log(got["prob"]), -loss.cpu().numpy(), atol=tol)


def test_other_stream_and_graph(torch, ctx):
    """A side stream, and two captured graphs with their own workspaces
    replayed on two streams at once with new inputs, give the eager bits."""
    N, V, D = 150, 3000, 128
    h, w, t, g = H.head_inputs(N, V, D, seed=13, device="cuda")

    def step():
        loss, lse = ctx.head_loss(h, w, t)
        dh, dw = ctx.head_loss_grad(h, w, t, lse, g)
        q, s = ctx.quantize_fp8(h)
        wq, ws = ctx.quantize_fp8(w, block_rows=128)
        return loss, lse, dh, dw, q.view(torch.uint8), s, ctx.matmul_fp8(q, s, wq, ws)

    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # an explicit stream handle
    loss, lse = ctx.head_loss(h, w, t, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step()
        graphs.append((gr, outs))
    h2 = H.head_inputs(N, V, D, seed=14, device="cuda")[0]
    h.copy_(h2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    ctx.poll_status()
    want = step()
    for _, outs in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


# ---------------------------------------------------------------- refusals
def test_refusals(torch, ctx):
    import ctypes

    from qwenium_b200 import qsamp

    h, w, t, g = H.head_inputs(8, 64, 32, device="cuda")
    bad = pytest.raises(qsamp.QsampError, match="expected")
    with bad:
        ctx.head_loss(h.float(), w, t)
    with bad:
        ctx.head_loss(h.cpu(), w, t)
    with bad:
        ctx.head_loss(h, w[:, :24], t)
    with bad:
        ctx.head_loss(h, w, t.long())
    with bad:
        ctx.head_loss(h, w, t[:4])
    with bad:
        ctx.head_loss(h.t(), w.t(), t)
    for cap in (-1.0, float("nan"), float("inf"), 1e-30, 1e30):
        with bad:
            ctx.head_loss(h, w, t, softcap=cap)
    with pytest.raises(qsamp.QsampError, match="multiple of 8") as e:
        ctx.head_loss(h[:, :20], w[:, :20], t)
    assert e.value.status == 3
    with pytest.raises(qsamp.QsampError, match="16-byte"):
        ctx.head_loss(h[:, 4:28], w[:, 4:28], t)
    lse = torch.zeros(8, device="cuda")
    with bad:
        ctx.head_loss_grad(h, w, t, lse[:4], g)
    with bad:
        ctx.head_loss_grad(h, w, t, lse, g, d_weight=torch.empty((64, 24), dtype=torch.bfloat16, device="cuda"))
    # a workspace too small, missing, or off its boundary
    head = ctx._head(h, w, t, 0.0)
    out = torch.empty(16, device="cuda")
    need = ctx.lib.qsamp_head_workspace(ctx.h, 8, 64, 32, 0)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    for ptr, n in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 16, need)):
        rc = ctx.lib.qsamp_head_loss(ctx.h, ctypes.byref(head), out.data_ptr(), out[8:].data_ptr(), ptr, n, None)
        assert rc == 1, (ptr, n)
    x, sx, wq, sw = H.fp8_inputs(4, 200, 48, device="cuda")
    with bad:
        ctx.matmul_fp8(x, sx[:2], wq, sw)
    with bad:
        ctx.matmul_fp8(x, sx, wq, sw[:1])
    with bad:
        ctx.matmul_fp8(x.float(), sx, wq, sw)
    with bad:
        ctx.matmul_fp8(x, sx, wq, sw, out=torch.empty((4, 200), dtype=torch.float16, device="cuda"))
    with pytest.raises(qsamp.QsampError, match="multiple of 16"):
        ctx.matmul_fp8(x[:, :40], sx, torch.zeros((200, 40), dtype=torch.uint8, device="cuda").view(x.dtype), sw)
    with bad:
        ctx.quantize_fp8(h, block_rows=64)
    with bad:
        ctx.quantize_fp8(h.half())


def test_workspace_of_refused_sizes(torch, ctx):
    """Sizes no call serves, whose workspace would not fit its 64 bits either."""
    size = lambda *a: ctx.lib.qsamp_head_workspace(ctx.h, *a)
    top = 2**31 - 1
    for grad in (0, 1):
        for n, v, d in ((-1, 8, 8), (1, 0, 8), (1, 8, 0), (top, top, top), (top, 8, 8), (1, top, 8), (1, 8, top),
                        (2**30, 8, 2**30), (8, 2**30, 2**30), (2**30, 2**30, 8)):
            assert size(n, v, d, grad) == -1, (n, v, d, grad)
        assert size(0, 8, 8, grad) >= 0 and size(2**22, 151936, 4096, grad) > 0
