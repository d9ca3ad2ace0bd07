"""The training operators run one after the other as a step uses them: norm (residual added) -> loss -> gradients of
loss and norm -> clipping of all gradients, against the same step in fp64 with torch's autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_head_of_a_model(ctx):
    T, V, D, eps = 400, 3001, 320, 1e-5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((T, D), generator=g, device="cuda").to(torch.bfloat16)
    res = torch.randn((T, D), generator=g, device="cuda").to(torch.bfloat16)
    wn = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
    w = (0.05 * torch.randn((V, D), generator=g, device="cuda")).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g, device="cuda")
    t[::7] = -100

    y, h = torch.empty_like(x), torch.empty_like(x)
    loss, lse, total = torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty(2, device="cuda")
    dy, dw, dx = torch.empty_like(x), torch.empty_like(w), torch.empty_like(x)
    dwn, norm = torch.empty(D, device="cuda"), torch.empty(1, device="cuda")
    clipped = [torch.empty((V, D), device="cuda"), torch.empty(D, device="cuda")]

    def step(stream):
        ctx.rmsnorm(x, wn, y, eps, residual=res, residual_out=h, stream=stream)
        ctx.linear_xent(y, w, t, loss, lse, total, stream=stream)
        ctx.linear_xent_backward(y, w, t, lse, dy, dw, total=total, stream=stream)
        ctx.rmsnorm_backward(dy, h, wn, dx, dwn, eps, stream=stream)
        ctx.grad_clip([dw, dwn], 0.01, norm, outs=clipped, stream=stream)

    step(None)
    ctx.sync()
    outs = [y, h, loss, total, dx, dwn, norm] + clipped
    eager = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager))

    h64 = (x.double() + res.double()).requires_grad_()
    wn64, w64 = wn.double().requires_grad_(), w.double().requires_grad_()
    y64 = h64 / torch.sqrt((h64 * h64).mean(dim=1, keepdim=True) + eps) * wn64
    want = torch.nn.functional.cross_entropy(y64 @ w64.T, t, ignore_index=-100)
    want.backward()
    want = want.detach()
    n64 = float(torch.sqrt(w64.grad.square().sum() + wn64.grad.square().sum()))
    # Every intermediate result (h, y, dy, dw) is rounded to bf16 once, 2^-8 of an element at most; a chain of four
    # such roundings stays under 4 * 2^-8 of a norm as long as no sum cancels, which these random ones do not.
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())   # noqa: E731
    assert abs(float(total[0] / total[1]) - float(want)) <= 2.0 ** -8 * float(want)
    assert rel(dx, h64.grad) <= 2.0 ** -6 and rel(dwn, wn64.grad) <= 2.0 ** -6 and rel(dw, w64.grad) <= 2.0 ** -6
    assert abs(float(norm) - n64) <= 2.0 ** -6 * n64
    assert rel(clipped[0], w64.grad * (0.01 / n64)) <= 2.0 ** -5 and rel(clipped[1], wn64.grad * (0.01 / n64)) <= 2.0 ** -5
