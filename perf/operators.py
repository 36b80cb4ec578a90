"""The output-head operators as they are measured: cases, inputs, plain forms.

Around the token selection stand the operators that make the logits and learn
from them: the head's product in 8-bit floating point with its quantisation
(serving), and the softmax cross entropy of head outputs over the whole
vocabulary with its gradients (scoring and training), which never holds the
[N, V] logits of all pieces at once. With ``own`` false ``run`` computes them
from elementary torch operations in 32 bits; with ``own`` true it makes the
calls of ``qwenium_b200.qsamp.Context``.

Formulas (h: hidden rows, w: head rows, t: targets, c: soft-cap, 0 for none):
  z[n,v]  = sum_d h[n,d] w[v,d];  l = z, or c tanh(z / c)
  lse[n]  = log sum_v exp l[n,v];  loss[n] = lse[n] - l[n,t[n]], 0 where t < 0
  dz[n,v] = g[n] (exp(l - lse) - [v = t[n]]) (1 - (l / c)^2 with a soft-cap), 0 where t < 0
  dh = dz w,  dw = dz^T h
  q, s    = a block's values over its scale s = amax / 448, rounded to e4m3
  out     = sum over blocks of 128 of sx sw (sum in the block of x w)
"""
import functools
import math

import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the log-probability of one generated token (a score request of one row)
        {"name": "score_one", "op": "score", "n": 1, "d": 1024, "v": 151936, "cap": 0.0, "ignored": 0.0},
        # a decode batch of 256 rows scored under a soft-capped head over the larger vocabulary
        {"name": "score_cap_256", "op": "score", "n": 256, "d": 2048, "v": 262144, "cap": 30.0, "ignored": 0.0},
        # a small fine-tuning step on a pruned vocabulary: odd rows, odd vocabulary, a third of the rows prompt tokens without a loss
        {"name": "train_ragged_509", "op": "train", "n": 509, "d": 1152, "v": 50021, "cap": 30.0, "ignored": 0.35},
        # a training step of a draft head: 4096 tokens
        {"name": "train_4096", "op": "train", "n": 4096, "d": 2048, "v": 151936, "cap": 0.0, "ignored": 0.1},
        # the largest: 8192 tokens of a wide model
        {"name": "train_8192", "op": "train", "n": 8192, "d": 4096, "v": 151936, "cap": 0.0, "ignored": 0.0},
        # the activations of a decode batch of ten slots before the 8-bit head
        {"name": "quant_rows_10", "op": "quant", "n": 10, "d": 4096, "rows": 1, "f32": False},
        # the activations of a long prompt, a width that ends inside a block
        {"name": "quant_rows_8000", "op": "quant", "n": 8000, "d": 8136, "rows": 1, "f32": False},
        # the head's own weights, laid out once when a server loads them
        {"name": "quant_head", "op": "quant", "n": 151936, "d": 4096, "rows": 128, "f32": False},
        # a single slot's decode step through the 8-bit head
        {"name": "fp8_one", "op": "fp8", "n": 1, "d": 4096, "v": 151936, "f32": False},
        # the ten slots of the server, fp32 logits for the sampler, a vocabulary without padding
        {"name": "fp8_10", "op": "fp8", "n": 10, "d": 2048, "v": 151655, "f32": True},
        # the headline batch of 256 rows
        {"name": "fp8_256", "op": "fp8", "n": 256, "d": 4096, "v": 151936, "f32": False},
        # a prompt's rows through a wide projection, a depth that ends inside a block
        {"name": "fp8_prompt_4096", "op": "fp8", "n": 4096, "d": 4048, "v": 16384, "f32": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "train", "quant", "fp8"])
    if op == "quant":
        rows = rng.choice([1, 1, 128])
        n = _log(rng, 1, 16384) if rows == 1 else _log(rng, 200, 151936)
        return {"op": op, "n": n, "d": 16 * _log(rng, 32, 512), "rows": rows, "f32": rng.random() < 0.25}
    if op == "fp8":
        n = _log(rng, 1, 4096)
        v = _log(rng, 2048, 262144 if n <= 512 else 16384)
        return {"op": op, "n": n, "d": 16 * _log(rng, 32, 256), "v": v, "f32": rng.random() < 0.4}
    n = _log(rng, 1, 1024 if op == "score" else 4096)
    v = _log(rng, 8192, 262144 if n <= 2048 else 151936)
    d = 8 * _log(rng, 64, 512 if n <= 2048 else 256)
    return {"op": op, "n": n, "d": d, "v": v, "cap": rng.choice([0.0, 0.0, 30.0]), "ignored": rng.choice([0.0, 0.2])}


# ---------------------------------------------------------------- inputs
def _scale_blocks(x, rows, blk):
    """amax over blocks of `rows` x BLOCK elements of x [n][d]; zero padding at the ends."""
    n, d = x.shape
    x = torch.nn.functional.pad(x, (0, -d % blk, 0, -n % rows))
    return x.abs().reshape(x.shape[0] // rows, rows, x.shape[1] // blk, blk).amax(dim=(1, 3))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape, dtype=torch.bfloat16, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    n, d = case["n"], case["d"]
    if case["op"] == "quant":
        # activations: unit rows with a few wide channels, as after a norm; weights: a plain normal
        x = torch.randn((n, d), generator=g, device=dev, dtype=torch.float32)
        if case["rows"] == 1:
            x *= torch.exp(0.5 * torch.randn((1, d), generator=g, device=dev))
        else:
            x *= d**-0.5
        return {"case": case, "x": x if case["f32"] else x.to(torch.bfloat16)}
    v = case["v"]
    if case["op"] == "fp8":
        x = randn(n, d, dtype=torch.float32)
        w = randn(v, d, dtype=torch.float32, scale=3.0 * d**-0.5)
        kb = -(-d // BLOCK)
        sx = _scale_blocks(x, 1, BLOCK) / E4M3_MAX
        sw = _scale_blocks(w, BLOCK, BLOCK) / E4M3_MAX
        xq = (x / sx.repeat_interleave(BLOCK, 1)[:, :d]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        w /= sw.repeat_interleave(BLOCK, 0)[:v].repeat_interleave(BLOCK, 1)[:, :d]
        wq = w.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        assert sx.shape == (n, kb)
        return {"case": case, "x": xq, "sx": sx, "w": wq, "sw": sw}
    w = randn(v, d, scale=3.0 * d**-0.5)
    t = torch.randint(0, v, (n,), generator=g, device=dev)
    # rows lean towards their target by a different amount each, as a partly trained model's do
    lean = torch.rand((n, 1), generator=g, device=dev) * 1.5
    h = (torch.randn((n, d), generator=g, device=dev) + lean * w[t].float()).to(torch.bfloat16)
    out = torch.rand((n,), generator=g, device=dev) < case["ignored"]
    t = torch.where(out, torch.full_like(t, -100), t).to(torch.int32)
    # the mean over the rows that have a loss
    gl = torch.ones((n,), device=dev) / (t >= 0).sum().clamp(min=1)
    return {"case": case, "h": h, "w": w, "t": t, "g": gl}


# ---------------------------------------------------------------- one pass
@functools.lru_cache(maxsize=None)
def _ctx(device):
    from qwenium_b200 import qsamp

    return qsamp.Context(device)


def run(state):
    c = state["case"]
    if own:
        ctx = _ctx(0)
        if c["op"] == "quant":
            return ctx.quantize_fp8(state["x"], block_rows=c["rows"])
        if c["op"] == "fp8":
            return ctx.matmul_fp8(state["x"], state["sx"], state["w"], state["sw"],
                                  out_dtype=torch.float32 if c["f32"] else torch.bfloat16)
        loss, lse = ctx.head_loss(state["h"], state["w"], state["t"], softcap=c["cap"])
        if c["op"] == "score":
            return loss, lse
        dh, dw = ctx.head_loss_grad(state["h"], state["w"], state["t"], lse, state["g"], softcap=c["cap"])
        return loss, lse, dh, dw
    if c["op"] == "quant":
        return _quant(state["x"], c["rows"])
    if c["op"] == "fp8":
        x = _dequant(state["x"], state["sx"], 1)
        out = x @ _dequant(state["w"], state["sw"], BLOCK).t()
        return out if c["f32"] else out.to(torch.bfloat16)
    return _loss(state, c["cap"], c["op"] == "train")


def _spread(s, rows, n, d):
    """A scale per block as a scale per element [n][d]."""
    return s.repeat_interleave(rows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :d]


def _dequant(q, s, rows):
    return q.float() * _spread(s, rows, *q.shape)


def _quant(x, rows):
    n, d = x.shape
    s = _scale_blocks(x.float(), rows, BLOCK)
    s = s / torch.full_like(s, E4M3_MAX)  # a tensor's quotient is rounded once; a number's is a product with its reciprocal
    # in 64 bits next to the borders between two e4m3 values; ties to even
    y = x.double()
    y = torch.where(x == 0, 0.0, y / _spread(s, rows, n, d).double()).clamp_(-E4M3_MAX, E4M3_MAX)
    e = torch.frexp(y.abs())[1].sub_(1).clamp_(min=-6).sub_(3)
    step = torch.ldexp(torch.ones_like(y), e)
    return (torch.round(y / step) * step).to(torch.float8_e4m3fn), s


def _loss(state, cap, grad):
    h, w, t = state["h"].float(), state["w"].float(), state["t"].long()
    z = h @ w.t()
    if cap > 0:
        z = torch.tanh(z / cap) * cap
    m = z.amax(dim=1, keepdim=True)
    # the sum of up to 262144 terms in 64 bits
    lse = m + torch.log(torch.exp(z - m).sum(dim=1, keepdim=True, dtype=torch.float64)).float()
    live = (t >= 0).unsqueeze(1)
    at = t.clamp(min=0).unsqueeze(1)
    loss = torch.where(live, lse - z.gather(1, at), 0.0)
    if not grad:
        return loss.squeeze(1), lse.squeeze(1)
    dz = torch.exp(z - lse)
    dz.scatter_add_(1, at, torch.full_like(lse, -1.0))
    if cap > 0:
        dz *= 1.0 - (z / cap) ** 2
    del z
    dz *= torch.where(live, state["g"].unsqueeze(1), 0.0)
    return loss.squeeze(1), lse.squeeze(1), (dz @ w).to(torch.bfloat16), (dz.t() @ h).to(torch.bfloat16)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, d = case["n"], case["d"]
    if case["op"] == "quant":
        blocks = -(-n // case["rows"]) * -(-d // BLOCK)
        return {"bytes": n * d * ((4 if case["f32"] else 2) + 1) + 4 * blocks, "flops": 2 * n * d}
    v = case["v"]
    if case["op"] == "fp8":
        kb = -(-d // BLOCK)
        scales = 4 * kb * (n + -(-v // BLOCK))
        return {"bytes": (n + v) * d + scales + n * v * (4 if case["f32"] else 2), "flops": 2 * n * v * d}
    one = {"bytes": 2 * (n + v) * d + 12 * n, "flops": 2 * n * v * d}
    if case["op"] == "score":
        return one
    return {"bytes": 4 * (n + v) * d + 16 * n, "flops": 6 * n * v * d}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quant":
        x, rows = st["x"], case["rows"]
        n, d = x.shape
        qs, ss = [], []
        for r in range(0, n, 4096):  # a multiple of 128 rows at a time
            p = x[r:r + 4096].double()
            s = torch.nn.functional.max_pool2d(p.abs()[None], (rows, BLOCK), ceil_mode=True)[0]
            s = s / torch.full_like(s, E4M3_MAX)
            s32 = s.float()  # the scale is what the call returns, in 32 bits
            y = p / s32.double().repeat_interleave(rows, 0)[:p.shape[0]].repeat_interleave(BLOCK, 1)[:, :d]
            y = torch.nan_to_num(y, nan=0.0).clamp_(-E4M3_MAX, E4M3_MAX)
            # the nearest of the 127 magnitudes, ties to the one with an even code
            grid = torch.arange(127, device=p.device, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).double()
            mid = (grid[1:] + grid[:-1]) / 2
            a = y.abs()
            lo = torch.searchsorted(mid, a, right=False)
            hi = torch.searchsorted(mid, a, right=True)
            code = torch.where(lo == hi, lo, torch.where(lo % 2 == 0, lo, hi))
            qs.append((grid[code] * torch.sign(y)).float())
            ss.append(s)
        return torch.cat(qs), torch.cat(ss)
    if case["op"] == "fp8":
        n, d = st["x"].shape
        x = st["x"].double() * st["sx"].double().repeat_interleave(BLOCK, 1)[:, :d]
        outs = []
        for r in range(0, case["v"], 8192):
            w = st["w"][r:r + 8192].double()
            s = st["sw"][r // BLOCK:(r + 8192) // BLOCK].double()
            outs.append(x @ (w * s.repeat_interleave(BLOCK, 0)[:w.shape[0]].repeat_interleave(BLOCK, 1)[:, :d]).t())
        return torch.cat(outs, dim=1)
    h, w, t, cap = st["h"].double(), st["w"].double(), st["t"].long(), case["cap"]
    n = h.shape[0]
    losses, lses, dhs = [], [], []
    dw = torch.zeros_like(w)
    for r in range(0, n, 2048):
        hr, tr = h[r:r + 2048], t[r:r + 2048]
        z = hr @ w.t()
        slope = 1.0
        if cap > 0:
            y = torch.tanh(z / cap)
            z, slope = y * cap, 1.0 - y * y
        lse = torch.logsumexp(z, dim=1)
        has = torch.nonzero(tr >= 0).squeeze(1)
        loss = torch.zeros_like(lse)
        loss[has] = lse[has] - z[has, tr[has]]
        losses.append(loss)
        lses.append(lse)
        if case["op"] == "train":
            p = torch.exp(z - lse.unsqueeze(1))
            p[has, tr[has]] -= 1.0
            keep = torch.zeros_like(lse)
            keep[has] = st["g"][r:r + 2048].double()[has]
            p = p * slope * keep.unsqueeze(1)
            dhs.append(p @ w)
            dw += p.t() @ hr
    if case["op"] == "score":
        return torch.cat(losses), torch.cat(lses)
    return torch.cat(losses), torch.cat(lses), torch.cat(dhs), dw
