"""Softmax cross entropy of a linear output layer (logits not kept) and its gradients against 64-bit forms.

Bars, per element, from the arithmetic.  Products of bf16 are exact in fp32; the tensor cores add them 16 at a
time and may cut a sum off instead of rounding it, 2^-23 of the sum of magnitudes per addition: a logit is within
d = (D / 16 + 16) 2^-23 max_v sum |h w|.  lse moves by at most d, and its exponentials and sums add 2^-20; the loss
takes 2 d + 2^-20 (1 + |lse|).  G's entries are p (relative 2 d + 2^-19) less the one at the target, rounded to bf16
(2^-8 of the entry): their errors reach dH through |W| and dW through |H|, the fp32 sums add 2^-16 of the sums
of magnitudes (K / 16 additions of up to 2^-23, K <= 2048), and the result is rounded once more, 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100
# (T, V, D, share of ignored tokens, elements between rows)
SHAPES = [(1, 1000, 128, 0.0, 0), (1, 1, 1, 0.0, 0), (5, 7, 8, 0.2, 0), (64, 256, 64, 0.0, 0), (256, 256, 64, 0.0, 8),
          (257, 257, 65, 0.3, 0), (300, 1021, 256, 0.1, 0), (130, 513, 100, 0.5, 3), (17, 300, 1, 0.0, 0), (17, 300, 33, 0.3, 2),
          (1000, 2000, 512, 0.6, 0), (3, 70000, 16, 0.0, 0), (2000, 129, 24, 0.05, 0)]


def make(T, V, D, ignored, pad, seed, std=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn((T, D + pad), generator=g, device="cuda").to(torch.bfloat16)[:, :D]
    w = (std * torch.randn((V, D + pad), generator=g, device="cuda")).to(torch.bfloat16)[:, :D]
    t = torch.randint(0, V, (T,), generator=g, device="cuda")
    t[torch.randperm(T, generator=g, device="cuda")[: int(T * ignored)]] = IGNORE
    return h, w, t, torch.rand(T, generator=g, device="cuda") + 0.25


class Reference:
    def __init__(self, h, w, t, weights):
        self.keep = (t != IGNORE) & (t >= 0) & (t < w.shape[0])
        h, w, t, g = h[self.keep].double(), w.double(), t[self.keep], weights[self.keep].double()
        self.n = len(t)
        at = torch.arange(self.n, device="cuda")
        logits = h @ w.T
        self.lse = torch.logsumexp(logits, dim=1)
        self.loss = self.lse - logits[at, t]
        self.d = (h.abs() @ w.abs().T).amax() * (h.shape[1] / 16 + 16) * 2.0 ** -23 if self.n else logits.new_zeros(())
        self.loss_bar = 2 * self.d + 2.0 ** -20 * (1 + self.lse.abs())
        p = torch.exp(logits - self.lse[:, None])
        G = p.clone()
        G[at, t] -= 1.0
        off = p * (2 * self.d + 2.0 ** -19) + G.abs() * 2.0 ** -8
        G, off = G * g[:, None], off * g[:, None]
        self.dh, self.dw = G @ w, G.T @ h
        self.dh_bar = off @ w.abs() + G.abs() @ w.abs() * 2.0 ** -16 + self.dh.abs() * 2.0 ** -8 + 1e-30
        self.dw_bar = off.T @ h.abs() + G.abs().T @ h.abs() * 2.0 ** -16 + self.dw.abs() * 2.0 ** -8 + 1e-30


def forward(ctx, h, w, t, **kw):
    loss, lse = torch.full((h.shape[0],), 9.0, device="cuda"), torch.full((h.shape[0],), 9.0, device="cuda")
    total = torch.full((2,), 9.0, device="cuda")
    ctx.linear_xent(h, w, t, loss, lse, total, ignore_index=IGNORE, **kw)
    return loss, lse, total


def within(got, want, bar):
    off = (got.double() - want).abs()
    assert bool((off <= bar).all()), float((off - bar).max())


@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(ctx, shape):
    T, V, D, ignored, pad = shape
    h, w, t, g = make(*shape, seed=T + V + D)
    ref = Reference(h, w, t, g)
    loss, lse, total = forward(ctx, h, w, t)
    dh = torch.full((T, D + pad), 5.0, dtype=torch.bfloat16, device="cuda")[:, :D]
    dw = torch.full((V, D + pad), 5.0, dtype=torch.bfloat16, device="cuda")[:, :D]
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE)
    ctx.sync()
    within(lse[ref.keep], ref.lse, ref.loss_bar)
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    assert bool((loss[~ref.keep] == 0).all()) and bool((lse[~ref.keep] == 0).all())
    assert float(total[1]) == ref.n
    assert abs(float(total[0]) - float(ref.loss.sum())) <= float(ref.loss_bar.sum()) + 2.0 ** -24 * float(ref.loss.sum().abs())
    within(dh[ref.keep], ref.dh, ref.dh_bar)
    assert bool((dh[~ref.keep] == 0).all())
    within(dw, ref.dw, ref.dw_bar)
    # the columns between the rows were left as they were
    if pad:
        assert bool((dh.as_strided((T, pad), (D + pad, 1), D)[:-1] == 5.0).all())
        assert bool((dw.as_strided((V, pad), (D + pad, 1), D)[:-1] == 5.0).all())


@pytest.mark.parametrize("shape", [(300, 1021, 256, 0.1, 0), (130, 513, 100, 0.5, 3)])
def test_gradient_of_the_mean(ctx, shape):
    h, w, t, _ = make(*shape, seed=3)
    loss, lse, total = forward(ctx, h, w, t)
    n = int((t != IGNORE).sum())
    ref = Reference(h, w, t, torch.full((shape[0],), 0.5 / n, device="cuda"))
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, total=total, ignore_index=IGNORE, scale=0.5)
    only_h, only_w = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, only_h, None, total=total, ignore_index=IGNORE, scale=0.5)
    ctx.linear_xent_backward(h, w, t, lse, None, only_w, total=total, ignore_index=IGNORE, scale=0.5)
    ctx.sync()
    within(dh[ref.keep], ref.dh, ref.dh_bar)
    within(dw, ref.dw, ref.dw_bar)
    assert torch.equal(dh, only_h) and torch.equal(dw, only_w)


def test_gradient_against_differences(ctx):
    """The mean loss of inputs a step of bf16 apart along a random direction: its change is the mean of the two ends'
    gradients along the step up to third order.  The step (2^-4 of each element, 16 elements moved per row) keeps that
    under 1 % of the change; the losses' rounding (2^-20 of 7 per token) is far below."""
    h, w, t, _ = make(64, 1000, 64, 0.0, 0, seed=8)
    to = h.clone()
    to[:, :16] = (h[:, :16].float() * (1 + 2.0 ** -4)).to(torch.bfloat16)
    sums, grads = [], []
    for x in (h, to):
        loss, lse, total = forward(ctx, x, w, t)
        dh = torch.empty_like(x)
        ctx.linear_xent_backward(x, w, t, lse, dh, None, dloss=torch.ones(64, device="cuda"), ignore_index=IGNORE)
        sums.append(float(loss.double().sum()))
        grads.append(dh.double())
    move = to.double() - h.double()
    along = float(((grads[0] + grads[1]) / 2 * move).sum())
    size = float(((grads[0].abs() + grads[1].abs()) / 2 * move.abs()).sum())
    assert abs((sums[1] - sums[0]) - along) <= 0.01 * size


def test_ignored_rows_may_hold_anything(ctx):
    h, w, t, g = make(200, 700, 72, 0.4, 0, seed=9)
    clean = h.clone()
    clean[t == IGNORE] = 0.0
    h[t == IGNORE] = float("nan")
    h[int(torch.nonzero(t == IGNORE)[0])] = float("inf")
    g[t == IGNORE] = float("nan")
    outs = []
    for x, gg in ((h, g), (clean, torch.nan_to_num(g))):
        loss, lse, total = forward(ctx, x, w, t)
        dh, dw = torch.empty_like(x), torch.empty_like(w)
        ctx.linear_xent_backward(x, w, t, lse, dh, dw, dloss=gg, ignore_index=IGNORE)
        ctx.sync()
        outs.append((loss, lse, total, dh, dw))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_no_token_counts(ctx):
    h, w, t, g = make(70, 300, 40, 1.0, 0, seed=10)
    # scratch that a counted call left NaN in
    bad = h.clone()
    bad[:] = float("nan")
    forward(ctx, bad, w, torch.zeros_like(t))
    loss, lse, total = forward(ctx, h, w, t)
    dh, dw = torch.full_like(h, 3.0), torch.full_like(w, 3.0)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, total=total, ignore_index=IGNORE)
    ctx.sync()
    for x in (loss, lse, total, dh, dw):
        assert bool((x == 0).all())
    empty = torch.empty((0, 40), dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    total.fill_(5.0)
    dw.fill_(3.0)
    ctx.linear_xent(empty, w, none, None, None, total)
    ctx.linear_xent_backward(empty, w, none, torch.empty(0, device="cuda"), None, dw, total=total)
    ctx.sync()
    assert bool((total == 0).all()) and bool((dw == 0).all())


def test_targets_out_of_range_are_loud_and_harmless(ctx):
    h, w, t, g = make(50, 300, 40, 0.1, 0, seed=11)
    at = [int(i) for i in torch.nonzero(t != IGNORE)[:2]]
    t[at[0]], t[at[1]] = 300, -7
    ref = Reference(h, w, t, g)
    loss, lse, total = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE)
    ctx.sync()
    assert bool(loss[at].isnan().all()) and bool(lse[at].isnan().all()) and bool(total[0].isnan())
    assert float(total[1]) == ref.n
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    assert bool((dh[at] == 0).all())
    within(dw, ref.dw, ref.dw_bar)


def test_large_logits_and_classes_of_minus_infinity(ctx):
    """Logits of hundreds (exp overflows without the maximum), and classes switched off by -inf in W."""
    h, w, t, _ = make(40, 600, 64, 0.0, 0, seed=12, std=8.0)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[300:556, 0] = float("-inf")          # whole 128-column stretches of a tile
    t = t % 300
    ref = Reference(h, w[list(range(300)) + list(range(556, 600))], t, torch.ones(40, device="cuda"))
    loss, lse, _ = forward(ctx, h, w, t)
    ctx.sync()
    within(lse, ref.lse, ref.loss_bar)
    within(loss, ref.loss, ref.loss_bar)


@pytest.mark.parametrize("T,V,D", [(2048, 131072 + 300, 64), (600, 70001, 50)])
def test_several_pieces_of_the_vocabulary(ctx, T, V, D):
    """More classes than one piece of G holds, and rows of W that have to be packed (D = 50)."""
    h, w, t, g = make(T, V, D, 0.1, 0, seed=13)
    t[-1] = V - 1
    loss, lse, _ = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE)
    ctx.sync()
    ref = Reference(h, w, t, g)
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    # dH adds V / 16 products in a row in places: 2^-23 each, 2^-10 of the magnitudes at most
    size = ref.dh_bar + 2.0 ** -10 * ref.dh.abs().amax()
    within(dh[ref.keep], ref.dh, size)
    within(dw, ref.dw, ref.dw_bar)


def test_offsets_beyond_32_bits(ctx):
    V, D = 600000, 4096                     # 2.46e9 elements
    g = torch.Generator(device="cuda").manual_seed(14)
    w = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    for first in range(0, V, 100000):
        w[first:first + 100000] = 0.02 * torch.randn((100000, D), generator=g, device="cuda")
    h = torch.randn((8, D), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.tensor([0, 1, V - 1, V - 2, 524288, 300000, IGNORE, V - 1], device="cuda")
    loss, lse, total = forward(ctx, h, w, t)
    dw = torch.empty_like(w)
    dh = torch.empty_like(h)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, total=total, ignore_index=IGNORE)
    ctx.sync()
    keep = t != IGNORE
    hk = h[keep].double()
    logits = torch.cat([hk @ w[f:f + 100000].double().T for f in range(0, V, 100000)], dim=1)
    l64 = torch.logsumexp(logits, dim=1)
    within(loss[keep], l64 - logits[torch.arange(7, device="cuda"), t[keep]], 1e-4)
    rows = torch.tensor([0, 2, 300000, 524287, 524288, 524289, V - 2, V - 1], device="cuda")
    p = torch.exp(logits[:, rows] - l64[:, None])
    p -= (t[keep][:, None] == rows[None, :]).double()
    want = p.T @ hk / 7
    bar = (p.abs().T @ hk.abs()) / 7 * 2.0 ** -7 + want.abs() * 2.0 ** -8
    within(dw[rows], want, bar)


def test_same_bits_again_on_another_stream_and_in_a_graph(ctx):
    h, w, t, g = make(500, 5000, 192, 0.2, 0, seed=15)
    small = make(40, 600, 64, 0.0, 0, seed=16)

    def both(out, stream):
        ctx.linear_xent(h, w, t, out[0], out[1], out[2], ignore_index=IGNORE, stream=stream)
        ctx.linear_xent_backward(h, w, t, out[1], out[3], out[4], dloss=g, ignore_index=IGNORE, stream=stream)

    def fresh():
        return [torch.zeros(500, device="cuda"), torch.zeros(500, device="cuda"), torch.zeros(2, device="cuda"),
                torch.zeros_like(h), torch.zeros_like(w)]

    runs = []
    for stream in (None, torch.cuda.Stream()):
        out = fresh()
        torch.cuda.synchronize()
        both(out, stream)
        torch.cuda.synchronize()
        runs.append(out)
        forward(ctx, *small[:3])            # another shape in between, in the same scratch
    out = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(out, torch.cuda.current_stream())
    big = make(3000, 50000, 256, 0.0, 0, seed=17)
    loss, lse, _ = forward(ctx, *big[:3])   # grows the scratch; the graph keeps the one it was captured with
    ctx.linear_xent_backward(big[0], big[1], big[2], lse, torch.empty_like(big[0]), torch.empty_like(big[1]), dloss=big[3])
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    runs.append(out)
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_growing_inside_a_capture_is_refused():
    from gern_b200 import api
    fresh = api.Context(0)
    h, w, t, _ = make(64, 500, 64, 0.0, 0, seed=18)
    loss = torch.zeros(64, device="cuda")
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1.0
        with pytest.raises(api.GernB200Error) as e:
            fresh.linear_xent(h, w, t, loss, None, stream=torch.cuda.current_stream())
        x += 1.0
    assert e.value.code == -3 and "before the capture" in str(e.value)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 2.0).all())
    fresh.close()


def test_refusals(ctx):
    from gern_b200 import api
    h, w, t, g = make(32, 100, 64, 0.0, 0, seed=19)
    loss, lse, total = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    for kw in (dict(dloss=g, total=total), dict()):
        with pytest.raises(api.GernB200Error) as e:
            ctx.linear_xent_backward(h, w, t, lse, dh, dw, **kw)
        assert e.value.code == -1 and "either dloss" in str(e.value)
    for a, b in ((None, None), (h, dw), (dh, w)):
        with pytest.raises(api.GernB200Error) as e:
            ctx.linear_xent_backward(h, w, t, lse, a, b, dloss=g)
        assert e.value.code == -1
    with pytest.raises(api.GernB200Error):
        ctx.linear_xent(h, w, t, None, None, None)
    with pytest.raises(TypeError):
        ctx.linear_xent(h.float(), w, t, loss, lse)
    with pytest.raises(TypeError):
        ctx.linear_xent(h, w, t.int(), loss, lse)
    with pytest.raises(ValueError):
        ctx.linear_xent(h, w, t[:-1], loss, lse)
    ctx.sync()


@pytest.mark.parametrize("T", [1, 31, 32, 33, 128, 129, 255, 256, 300, 385, 1023, 1024, 1025, 8191, 8193])
@pytest.mark.parametrize("V", [200, 4100])
def test_every_number_of_tokens(ctx, T, V):
    """Around the borders of the tilings (32, 128, 256, 257 to 384 tokens), of the two ways of listing the counted
    tokens (1024) and of their steps (8192); with few classes and with enough for narrow tiles."""
    h, w, t, g = make(T, V, 40, 0.3, 0, seed=T)
    ref = Reference(h, w, t, g)
    loss, lse, total = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE)
    ctx.sync()
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    assert bool((loss[~ref.keep] == 0).all()) and float(total[1]) == ref.n
    # dW adds the tokens up: T / 16 additions of at most 2^-23 of the magnitudes beyond the 2^-16 of the bar
    within(dh[ref.keep], ref.dh, ref.dh_bar)
    within(dw, ref.dw, ref.dw_bar)


@pytest.mark.parametrize("D,ld", [(15, 16), (20, 24), (100, 104), (33, 40), (64, 72), (65, 72)])
@pytest.mark.parametrize("T", [14, 200])
def test_columns_between_rows_are_neither_read_nor_written(ctx, T, D, ld):
    """Rows that start on 16 bytes but end inside such a piece, NaN between them in the inputs; the results' last
    row ends where its buffer's guarded part begins."""
    V = 700
    h0, w0, t, g = make(T, V, D, 0.2, 0, seed=D)
    h = torch.full((T, ld), float("nan"), dtype=torch.bfloat16, device="cuda")
    w = torch.full((V, ld), float("nan"), dtype=torch.bfloat16, device="cuda")
    h[:, :D], w[:, :D] = h0, w0
    h, w = h[:, :D], w[:, :D]
    ref = Reference(h0, w0, t, g)
    loss, lse, _ = forward(ctx, h, w, t)
    bufs, outs = [], []
    for rows in (T, V):
        bufs.append(torch.full(((rows - 1) * ld + D + 40,), 5.0, dtype=torch.bfloat16, device="cuda"))
        outs.append(bufs[-1].as_strided((rows, D), (ld, 1)))
    ctx.linear_xent_backward(h, w, t, lse, outs[0], outs[1], dloss=g, ignore_index=IGNORE)
    ctx.sync()
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    within(outs[0][ref.keep], ref.dh, ref.dh_bar)
    within(outs[1], ref.dw, ref.dw_bar)
    for buf, out in zip(bufs, outs):
        outside = torch.ones_like(buf, dtype=torch.bool)
        outside.as_strided(out.shape, (ld, 1)).fill_(False)
        assert bool((buf[outside] == 5.0).all())


def test_scratch_that_cannot_be_had_is_an_error_and_no_more(ctx):
    """2^24 tokens over 2^26 classes would need 64 TiB for their maxima and sums; the context works on afterwards."""
    from gern_b200 import api
    h = torch.empty((1 << 24, 8), dtype=torch.bfloat16, device="cuda")
    w = torch.empty((1 << 26, 8), dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(1 << 24, dtype=torch.int64, device="cuda")
    with pytest.raises(api.GernB200Error) as e:
        ctx.linear_xent(h, w, t, None, None, torch.empty(2, device="cuda"))
    assert e.value.code == -2 and "scratch" in str(e.value)
    del h, w, t
    h, w, t, g = make(64, 300, 64, 0.1, 0, seed=20)
    ref = Reference(h, w, t, g)
    loss, lse, total = forward(ctx, h, w, t)
    ctx.sync()
    within(loss[ref.keep], ref.loss, ref.loss_bar)


@pytest.mark.parametrize("mean", [False, True])
def test_no_tokens_in_every_form(ctx, mean):
    """A batch without tokens: its per-token operands are empty tensors, which have no address.  dW is zeroed where it is
    wanted, its gaps are left, and a total is zeroed."""
    h = torch.empty((0, 40), dtype=torch.bfloat16, device="cuda")
    w = torch.randn((300, 40), device="cuda").to(torch.bfloat16)
    t, none = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda")
    total = torch.full((2,), 5.0, device="cuda")
    for loss, lse in ((none, none), (none, None), (None, none)):
        ctx.linear_xent(h, w, t, loss, lse)
    ctx.linear_xent(h, w, t, none, none, total)
    ctx.sync()
    assert bool((total == 0).all())
    room = torch.full((300, 48), 3.0, dtype=torch.bfloat16, device="cuda")
    kw = dict(total=total) if mean else dict(dloss=none)
    ctx.linear_xent_backward(h, w, t, none, torch.empty_like(h), None, **kw)
    for dh in (None, torch.empty_like(h)):
        room.fill_(3.0)
        ctx.linear_xent_backward(h, w, t, none, dh, room[:, :40], **kw)
        ctx.sync()
        assert bool((room[:, :40] == 0).all()) and bool((room[:, 40:] == 3.0).all())


@pytest.mark.parametrize("T", [5, 300, 1500])
@pytest.mark.parametrize("scale", [1.0, 4.0])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_a_weight_out_of_range_stays_in_its_row(ctx, T, scale, bad):
    """A token's infinite, NaN or huge dloss reaches its own row of dH and dW, and no other token's row of dH."""
    h, w, t, g = make(T, 200, 72, 0.2, 0, seed=21)
    at = int(torch.nonzero(t != IGNORE)[-1])
    ref = Reference(h, w, t, scale * g)
    g[at] = bad
    loss, lse, _ = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE, scale=scale)
    ctx.sync()
    others = torch.nonzero(ref.keep)[:, 0] != at
    within(dh[ref.keep][others], ref.dh[others], ref.dh_bar[others])
    assert bool((dh[~ref.keep] == 0).all())
    if bad != 3e38:
        assert not bool(torch.isfinite(dh[at]).any()) and not bool(torch.isfinite(dw).any())


def test_gradient_of_w_over_millions_of_tokens(ctx):
    """Sums over 2^22 tokens whose terms have one sign.  Logits are 0 and there are 8 classes, so G is exactly 1/8 (lse is
    within 2^-22, G rounds to bf16) and dW[v] the tokens' mean row over 8.  Bar: a product's sums are cut off at most
    1024 times in a row, 2^-24 of them on average and 2^-23 at most, 256 parts are added in fp32, the result is rounded."""
    T, V, D = 1 << 22, 8, 8
    g = torch.Generator(device="cuda").manual_seed(22)
    h = (0.5 + 0.5 * torch.rand((T, D), generator=g, device="cuda")).to(torch.bfloat16)
    w = torch.zeros((V, D), dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(T, dtype=torch.int64, device="cuda")
    lse, dw = torch.empty(T, device="cuda"), torch.empty_like(w)
    ctx.linear_xent(h, w, t, None, lse)
    ctx.linear_xent_backward(h, w, t, lse, None, dw, dloss=torch.ones(T, device="cuda"))
    ctx.sync()
    want = h.double().sum(dim=0) / 8
    bar = want * (2.0 ** -8 + 2.0 ** -13 + 2.0 ** -16)
    within(dw[1:], want.expand(V - 1, D), bar)
    within(dw[0], -7 * want, 7 * bar)


def test_gradient_of_h_over_a_long_vocabulary(ctx):
    """One range of 2^18 classes for every tile of dH, terms of one sign.  H is 0, so G is exactly 2^-18 beside the target's
    entry, whose row of W is 0, and every row of dH the mean row of W.  The mean of the signed relative errors over 9472
    columns of different sizes: roundings to bf16 (2^-9 and less each, as often up as down) leave 2^-9 / sqrt(9472) < 2^-15
    of it, the sums at most 1024 cuts of 2^-24 on average in a row, 2^-14."""
    T, V, D = 512, 1 << 18, 9472
    g = torch.Generator(device="cuda").manual_seed(23)
    size = torch.exp2(torch.rand(D, generator=g, device="cuda"))
    w = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    want = torch.zeros(D, dtype=torch.float64, device="cuda")
    for first in range(0, V, 1 << 14):
        part = w[first:first + (1 << 14)]
        part.copy_(torch.rand(part.shape, generator=g, device="cuda").square() * size)
        if first == 0:
            part[0] = 0.0
        want += part.double().sum(dim=0) / V
    h = torch.zeros((T, D), dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(T, dtype=torch.int64, device="cuda")
    lse, dh = torch.empty(T, device="cuda"), torch.empty_like(h)
    ctx.linear_xent(h, w, t, None, lse)
    ctx.linear_xent_backward(h, w, t, lse, dh, None, dloss=torch.ones(T, device="cuda"))
    ctx.sync()
    off = dh[0].double() / want - 1.0
    assert bool((dh == dh[0]).all()) and float(off.abs().max()) <= 2.0 ** -8 + 2.0 ** -13
    assert abs(float(off.mean())) <= 2.0 ** -13


def test_gradients_of_the_longest_rows(ctx):
    """Rows of 2^20 elements whose products have one sign (logits of 30).  The loss's product is cut off 64 times in a row
    at most and added up from 1024 parts in fp32, G's 256 times and from 256 parts, 2^-23 of the sum each cut, 2^-24 each
    addition: logits and lse are within d = 30 (2^-17 + 2^-14 + 2^-15 + 2^-16), and the bars of the gradients follow
    from that as above."""
    T, V, D = 3, 5, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(24)
    h = (0.5 + 0.5 * torch.rand((T, D), generator=g, device="cuda")).to(torch.bfloat16)
    w = ((0.5 + 0.5 * torch.rand((V, D), generator=g, device="cuda")) * (30 / 0.5625 / D)).to(torch.bfloat16)
    t = torch.tensor([0, 4, 2], device="cuda")
    loss, lse, _ = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=torch.ones(T, device="cuda"))
    ctx.sync()
    ref = Reference(h, w, t, torch.ones(T, device="cuda"))
    logits = h.double() @ w.double().T
    d = float(logits.max()) * (2.0 ** -17 + 2.0 ** -14 + 2.0 ** -15 + 2.0 ** -16)
    within(loss, ref.loss, 2 * d + 2.0 ** -20 * (1 + ref.lse.abs()))
    p = torch.exp(logits - ref.lse[:, None])
    G = p.clone()
    G[torch.arange(T, device="cuda"), t] -= 1.0
    off = p * (2 * d + 2.0 ** -19) + G.abs() * 2.0 ** -8
    within(dh, ref.dh, off @ w.double().abs() + G.abs() @ w.double().abs() * 2.0 ** -16 + ref.dh.abs() * 2.0 ** -8)
    within(dw, ref.dw, off.T @ h.double() + G.abs().T @ h.double() * 2.0 ** -16 + ref.dw.abs() * 2.0 ** -8)


@pytest.mark.parametrize("T", [1, 257])
def test_scratch_of_few_tokens_over_many_classes(ctx, T):
    """G takes 256 MiB and no more, whatever the number of classes; H, its sums and lists are small here."""
    from gern_b200 import api
    V, D = 1 << 21, 8
    h, w, t, g = make(T, V, D, 0.0, 0, seed=25)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    _, lse, _ = forward(ctx, h, w, t)
    ctx.linear_xent_backward(h[:1], w[:99], t[:1] % 99, lse[:1], dh[:1], dw[:99], dloss=g[:1])    # (loads the kernels)
    ctx.sync()
    fresh = api.Context(0)
    before = torch.cuda.mem_get_info()[0]
    fresh.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g)
    fresh.sync()
    taken = before - torch.cuda.mem_get_info()[0]
    fresh.close()
    assert taken <= (256 + 64) << 20, taken >> 20
    # dW's rows for the first tokens' target classes: g (p - 1) h where one token has that target
    logits = torch.cat([h.double() @ w[f:f + (1 << 18)].double().T for f in range(0, V, 1 << 18)], dim=1)
    l64 = torch.logsumexp(logits, dim=1)
    p = torch.exp(logits[:, t] - l64[:, None])
    p -= (t[:, None] == t[None, :]).double()
    G = p * g.double()[:, None]
    within(dw[t], G.T @ h.double(), (G.abs().T @ h.double().abs()) * 2.0 ** -6)


@pytest.mark.parametrize("T,V,D", [(20, 300, 40), (300, 300, 72)])
def test_gradients_beside_their_operands(ctx, T, V, D):
    """dH in the columns beside H and dW in those beside W: no byte is shared."""
    h, w, t, g = make(T, V, D, 0.2, 0, seed=26)
    tokens, classes = torch.full((T, 2 * D + 8), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((V, 2 * D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    tokens[:, :D], classes[:, :D] = h, w
    ref = Reference(h, w, t, g)
    loss, lse, _ = forward(ctx, tokens[:, :D], classes[:, :D], t)
    ctx.linear_xent_backward(tokens[:, :D], classes[:, :D], t, lse, tokens[:, D:2 * D], classes[:, D:2 * D], dloss=g, ignore_index=IGNORE)
    ctx.sync()
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    within(tokens[:, D:2 * D][ref.keep], ref.dh, ref.dh_bar)
    within(classes[:, D:2 * D], ref.dw, ref.dw_bar)
    assert torch.equal(tokens[:, :D], h) and torch.equal(classes[:, :D], w)
    assert bool((tokens[:, 2 * D:] == 5.0).all()) and bool((classes[:, 2 * D:] == 5.0).all())


@pytest.mark.parametrize("T,V,D", [(20, 500, 9000), (100, 300, 8192), (300, 300, 8200), (40000, 300, 40), (16500, 300, 4160), (100, 1 << 19, 1792)])
def test_sums_of_several_parts(ctx, T, V, D):
    """Sums that leave the tensor cores in parts, on every tiling: logits of more than 4096 products (G), tokens or classes
    of more than 16384 (dW; dH, whose classes are cut into ranges too), with ordinary items beside them."""
    h, w, t, g = make(T, V, D, 0.1, 0, seed=27, std=0.05)
    loss, lse, _ = forward(ctx, h, w, t)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, dh, dw, dloss=g, ignore_index=IGNORE)
    again, alone = torch.empty_like(h), torch.empty_like(w)
    ctx.linear_xent_backward(h, w, t, lse, again, alone, dloss=g, ignore_index=IGNORE)
    ctx.sync()
    assert torch.equal(dh, again) and torch.equal(dw, alone)
    ref = Reference(h, w, t, g)
    within(loss[ref.keep], ref.loss, ref.loss_bar)
    # up to 1024 additions of 2^-23 in a row instead of the bar's 128: 2^-13 of the sums of magnitudes
    keep = ref.keep
    p = torch.exp(h[keep].double() @ w.double().T - ref.lse[:, None])
    p[torch.arange(ref.n, device="cuda"), t[keep]] -= 1.0
    p = p.abs_().mul_(g[keep].double()[:, None])
    within(dh[keep], ref.dh, ref.dh_bar + p @ w.double().abs() * 2.0 ** -13)
    within(dw, ref.dw, ref.dw_bar + p.T @ h[keep].double().abs() * 2.0 ** -13)
