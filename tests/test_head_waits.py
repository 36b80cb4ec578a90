"""The bounded waits of the output-head kernels: what a wait that ran out does,
how it is reported, and that the next call is served."""
import pytest

import head_cases as H


def test_no_context():
    from qwenium_b200 import build as qbuild
    from qwenium_b200 import qsamp

    qbuild.build()
    assert qsamp.load().qsamp_set_head_wait(None, 1) == 1


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture
def ctx(torch):
    from qwenium_b200 import qsamp

    return qsamp.Context(0)


@pytest.mark.gpu
def test_refusal(ctx):
    from qwenium_b200 import qsamp

    with pytest.raises(qsamp.QsampError, match="ns: expected >= 0, got -1"):
        ctx.set_head_wait(-1)


# the kernels: few-row loss, dz, and their gradients' pair kernel; the pair's loss and dz; sums of several
# slices (35000 rows); the 8-bit product's two kernels
@pytest.mark.gpu
@pytest.mark.parametrize("op,N", [("loss", 20), ("loss", 300), ("grad", 20), ("grad", 300), ("grad", 35000), ("product", 20),
                                  ("product", 300)])
def test_a_wait_that_runs_out(torch, ctx, op, N):
    """No time to wait for the first copies: the kernels leave, the call's error is
    reported once, and the same call with time gives its results to the bit."""
    from qwenium_b200 import qsamp

    V, D = 1000, 1024
    if op == "product":
        args = H.fp8_inputs(N, V, D, device="cuda")
        call = lambda: (ctx.matmul_fp8(*args),)
    else:
        h, w, t, g = H.head_inputs(N, V, D, seed=22, device="cuda")
        lse = ctx.head_loss(h, w, t)[1]
        call = lambda: ctx.head_loss(h, w, t) if op == "loss" else ctx.head_loss_grad(h, w, t, lse, g)
    want = call()
    torch.cuda.synchronize()
    ctx.poll_status()
    ctx.set_head_wait(0)
    call()
    torch.cuda.synchronize()
    with pytest.raises(qsamp.QsampError, match="bounded wait ran out in an output-head kernel") as e:
        ctx.poll_status()
    assert e.value.status == 4
    ctx.poll_status()
    ctx.set_head_wait(2_000_000_000)
    got = call()
    torch.cuda.synchronize()
    ctx.poll_status()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_reported_before_the_selection(torch, ctx):
    """The output head's report comes first and once; the selection's own status stays."""
    import numpy as np

    from qwenium_b200 import qsamp
    from qwenium_b200 import workloads as W

    h, w, t, _ = H.head_inputs(10, 5000, 64, seed=23, device="cuda")
    ctx.set_head_wait(0)
    ctx.head_loss(h, w, t)
    logits = (h.float() @ w.float().t()).contiguous()
    ids = torch.empty(10, dtype=torch.int32, device="cuda")
    ctx.sample_batch(logits, W.default_params(10), u=np.linspace(0.05, 0.95, 10), out_ids=ids)
    torch.cuda.synchronize()
    with pytest.raises(qsamp.QsampError, match="output-head"):
        ctx.poll_status()
    ctx.poll_status()
    assert (ids >= 0).all()
