"""Inputs, 64-bit results and error bounds for the output-head operators.

Everything is plain torch on the CPU or the GPU; the product is not used. A
rounding to a type is off by at most half a step: U32 and U16 below, relative
to the value.
"""
import torch

U32 = 2.0**-24  # fp32, half a step
U16 = 2.0**-8  # bf16, half a step
BLOCK = 128


def bf16(x):
    return x.to(torch.bfloat16)


def head_inputs(N, V, D, seed=0, scale=3.0, ignored=0.2, device="cpu"):
    g = torch.Generator().manual_seed(seed * 7919 + N * 31 + V * 7 + D)
    h = bf16(torch.randn((N, D), generator=g))
    w = bf16(torch.randn((V, D), generator=g) * (scale / D**0.5))
    t = torch.randint(0, V, (N,), generator=g).to(torch.int32)
    if N:
        t[torch.rand((N,), generator=g) < ignored] = -100
        t[0] = V - 1
    if N > 2:
        t[1], t[2] = 0, -1
    grad = torch.randn((N,), generator=g)
    return tuple(x.to(device) for x in (h, w, t, grad))


def head_exact(h, w, t, grad, cap, dz_error=U16):
    """64-bit loss, lse, dh, dw and the bounds of the bf16 / fp32 results.

    Logits: a sum of D products in 32 bits, in any order, is off by at most
    D U32 sum |h w| (first order); the cap's slope is at most 1 and its own
    evaluation is off by at most 6 U32 of the cap (the exponential, the quotient,
    the difference), or with a cap above 64 by 32 U32 of the result: 22 where
    |z / cap| is 1/4, fewer above, 6 of the series below. lse: the logits' error, the
    exponentials (an argument rounded to U32 of at most 2^7, a 4 U32
    evaluation), sums of V terms in any order, one logarithm and the final
    rounding. dz is rounded to bf16; sums of the products in 32 bits;
    the results rounded to bf16. dz_error: dz's own rounding, U16 (few rows
    have it in two parts: U16 squared).
    """
    N, D = h.shape
    V = w.shape[0]
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    ez = (D + 8) * U32 * (hd.abs() @ wd.abs().t())
    slope = torch.ones_like(z)
    if cap > 0:
        y = torch.tanh(z / cap)
        z, slope = cap * y, 1 - y * y
        ez = ez + 32 * U32 * (z.abs() if cap > 64 else cap)
    lse = torch.logsumexp(z, dim=1) if N else z.new_zeros(0)
    elog = ez.amax(dim=1) if N else z.new_zeros(0)
    elsum = elog + (V + 2**8) * U32 + 4 * U32 * lse.abs()
    live = (t >= 0) & (t < V)
    at = t.long().clamp(0, V - 1).unsqueeze(1)
    tz = z.gather(1, at).squeeze(1)
    loss = torch.where(live, lse - tz, torch.where(t >= V, torch.nan, 0.0))
    eloss = elsum + ez.gather(1, at).squeeze(1) + 2 * U32 * (lse.abs() + tz.abs())
    p = torch.exp(z - lse.unsqueeze(1))
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    gr = torch.where(live, grad.double(), 0.0).unsqueeze(1)
    dz = (p - hot) * slope * gr
    # a logit off by e moves p by p e, and the cap's slope by 2 e / cap
    edz = dz_error * dz.abs() + gr.abs() * slope.abs() * p * (ez + elsum.unsqueeze(1) + 2**-16)
    edz = edz + gr.abs() * (p + hot) * 8 * U32
    if cap > 0:
        edz = edz + gr.abs() * (p + hot) * (2 * ez / cap + 8 * U32)
    dh, dw = dz @ wd, dz.t() @ hd
    edh = edz @ wd.abs() * (1 + 2 * U16) + (V + 64) * U32 * (dz.abs() @ wd.abs()) + U16 * dh.abs()
    edw = edz.t() @ hd.abs() * (1 + 2 * U16) + (N + 64) * U32 * (dz.abs().t() @ hd.abs()) + U16 * dw.abs()
    tiny = 2.0**-126
    return {"loss": loss, "lse": lse, "eloss": eloss, "else": elsum, "dh": dh, "dw": dw, "edh": edh + tiny,
            "edw": edw + tiny}


def quant_exact(x, rows):
    """Scales (fp32) and e4m3 values of x [M][K] (float32 / bfloat16) in
    blocks of rows x 128, each value the nearest of the format's (ties to an
    even code) to the quotient in 64 bits; as float64."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    mb = -(-M // rows)
    xd = x.double()
    grid = torch.arange(127, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).double()
    q = torch.zeros_like(xd)
    s = torch.zeros((mb, kb), dtype=torch.float32)
    for i in range(mb):
        for j in range(kb):
            b = xd[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK]
            if not torch.isfinite(b).all():
                s[i, j] = torch.nan
                q[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK] = torch.nan
                continue
            s[i, j] = (b.abs().max() / 448.0).float()
            y = torch.where(b == 0, 0.0, b / s[i, j].double()).clamp(-448.0, 448.0)
            d = (y.abs().reshape(-1, 1) - grid).abs()
            near = d.min(dim=1, keepdim=True).values
            cand = torch.nonzero(d == near)
            code = torch.zeros(d.shape[0], dtype=torch.long)
            for r, c in cand.tolist():
                code[r] = c if (d[r] == near[r]).sum() == 1 or c % 2 == 0 else code[r]
            q[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK] = (grid[code] * torch.sign(y.reshape(-1))).reshape(b.shape)
    return q, s


def fp8_inputs(M, V, K, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed * 104729 + M * 31 + V * 7 + K)
    kb = -(-K // BLOCK)
    x = (torch.randn((M, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (torch.randn((V, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sx = torch.exp(torch.randn((M, kb), generator=g)) / 300
    sw = torch.exp(torch.randn((-(-V // BLOCK), kb), generator=g)) / (300 * K**0.5)
    return tuple(t.to(device) for t in (x, sx, w, sw))


def fp8_exact(x, sx, w, sw):
    """64-bit product and the bound of its fp32 result: sums of 128 products
    and of the blocks in 32 bits in any order, the scales' product and its
    application two roundings more per block."""
    M, K = x.shape
    V = w.shape[0]
    xd = x.double() * sx.double().repeat_interleave(BLOCK, 1)[:, :K]
    wd = w.double() * sw.double().repeat_interleave(BLOCK, 0)[:V].repeat_interleave(BLOCK, 1)[:, :K]
    return xd @ wd.t(), (K + 8) * U32 * (xd.abs() @ wd.abs().t())
