"""RMS norm with the residual's addition, its e4m3 output and its backward pass against 64-bit forms.

Bars, per element, derived from the arithmetic: u = 2^-24 is half a step of fp32.  A thread adds at most
40 squares one after the other and the team's tree adds 10 levels, so the sum of squares is within 51u,
r within 26u plus rsqrt's 4u; two products more give less than 2^6 u = 2^-18 relative.  A result rounded to
bf16 adds half a step, 2^-8; to e4m3 2^-4 of the value, or 2^-10 of the scale below its smallest normal.
A gradient is a difference of two terms: its fp32 error is 2^-18 of the terms' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6
FP32 = 2.0 ** -18
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float32]
# (rows, cols, columns between a row's end and the next row's start): one row, rows of one column, odd widths
# (no vector loads), every team size, rows too long for registers
SHAPES = [(1, 4096, 0), (3, 1, 0), (5, 7, 2), (33, 510, 0), (17, 512, 8), (9, 1000, 3), (129, 1021, 0), (7, 2048, 1),
          (300, 4096, 0), (5, 4104, 8), (6, 8192, 0), (4, 8200, 0), (4, 9000, 0), (3, 16384, 0), (3, 16386, 0), (2, 20001, 0),
          (1, 40000, 0), (2051, 64, 0)]


def make(rows, cols, pad, dtype, seed, n=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = [torch.randn((rows, cols + pad), generator=g, device="cuda").to(dtype)[:, :cols] for _ in range(n)]
    return out + [(1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)]


def norm64(h, w):
    r = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    return h * r * w.double(), r


def close(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off - bound).max())} beyond the bar"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(ctx, shape, dtype):
    x, res, w = make(*shape, dtype, sum(shape), 2)
    y, h = torch.empty_like(x), torch.empty_like(x)
    ctx.rmsnorm(x, w, y, EPS, residual=res, residual_out=h)
    plain, kept = torch.empty_like(x), torch.empty_like(x)
    ctx.rmsnorm(x, w, plain, EPS)
    ctx.rmsnorm(x, w, kept, EPS, residual_out=kept.new_empty(kept.shape))
    ctx.sync()
    want, _ = norm64(x.double() + res.double(), w)
    close(y, want, want.abs() * (FP32 + HALF[dtype]) + 1e-30, "y")
    s = x.double() + res.double()
    close(h, s, s.abs() * (2 * HALF[dtype]), "h")
    want, _ = norm64(x.double(), w)
    close(plain, want, want.abs() * (FP32 + HALF[dtype]) + 1e-30, "y without residual")
    assert torch.equal(plain, kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_e4m3_output(ctx, shape, group, dtype):
    rows, cols, _ = shape
    x, res, w = make(*shape, dtype, 1 + sum(shape), 2)
    groups = -(-cols // group) if group else 1
    q = torch.empty((rows, cols + 5), dtype=torch.float8_e4m3fn, device="cuda")[:, :cols]
    scales = torch.empty((rows, groups), device="cuda")
    ctx.rmsnorm_e4m3(x, w, q, scales, EPS, group=group, residual=res)
    ctx.sync()
    want, _ = norm64(x.double() + res.double(), w)
    width = group or cols
    top = torch.stack([want[:, i * width:(i + 1) * width].abs().amax(dim=1) for i in range(groups)], dim=1)
    close(scales, top / 448.0, top / 448.0 * FP32 + 2.0 ** -126, "scales")
    s = scales.double().repeat_interleave(width, dim=1)[:, :cols]
    close(q.float().double() * s, want, torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -12), "q * scale")


# rows whose operands all lie on 16 or 32 bytes: parts of warps, warps, blocks of every size
GRID = [(131, 8), (77, 40), (130, 64), (67, 128), (5, 136), (66, 256), (9, 264), (33, 512), (9, 896), (10, 1024), (7, 1536), (6, 2048),
        (5, 2560), (4, 4096), (4, 4104), (3, 5120), (3, 8192), (2, 10240), (2, 12296), (2, 12304), (2, 16384)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [None, 0, 32, 64, 128])
@pytest.mark.parametrize("shape", GRID)
def test_rows_on_the_vectors_grid(ctx, shape, group, dtype):
    """group None: the plain norm.  residual_out lies on x; the rows behind the last stay as they were."""
    rows, cols = shape
    x, res, w = make(rows, cols, 0, dtype, 5 + rows + cols, 2)
    s = x.double() + res.double()
    want, _ = norm64(s, w)
    room = torch.cat([x, torch.full_like(x[:2], 5.0)])
    if group is None:
        y = torch.full_like(room, 7.0)
        ctx.rmsnorm(room[:rows], w, y[:rows], EPS, residual=res, residual_out=room[:rows])
        ctx.sync()
        close(y[:rows], want, want.abs() * (FP32 + HALF[dtype]) + 1e-30, "y")
        assert bool((y[rows:] == 7.0).all())
    else:
        groups = -(-cols // group) if group else 1
        q = torch.full((rows + 2, cols), 1.5, device="cuda").to(torch.float8_e4m3fn)
        scales = torch.full((rows + 2, groups), 7.0, device="cuda")
        ctx.rmsnorm_e4m3(room[:rows], w, q[:rows], scales[:rows], EPS, group=group, residual=res, residual_out=room[:rows])
        ctx.sync()
        width = group or cols
        top = torch.stack([want[:, i * width:(i + 1) * width].abs().amax(dim=1) for i in range(groups)], dim=1)
        close(scales[:rows], top / 448.0, top / 448.0 * FP32 + 2.0 ** -126, "scales")
        each = scales[:rows].double().repeat_interleave(width, dim=1)[:, :cols]
        close(q[:rows].float().double() * each, want, torch.maximum(want.abs() * 2.0 ** -4, each * 2.0 ** -10) * (1 + 2.0 ** -12), "q * scale")
        assert bool((q[rows:].float() == 1.5).all()) and bool((scales[rows:] == 7.0).all())
    close(room[:rows], s, s.abs() * (2 * HALF[dtype]), "residual_out")
    assert bool((room[rows:] == 5.0).all())


@pytest.mark.parametrize("shape", [(5, 512, 0), (6, 1021, 0), (7, 4096, 0), (4, 4094, 1), (9, 40, 0), (3, 9000, 0)])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("sizes", [(1.0, 2.0 ** 102), (1.0, 2.0 ** -100), (2.0 ** -50, 1.0), (2.0 ** 55, 2.0 ** -20), (2.0 ** 40, 2.0 ** 90)])
def test_e4m3_of_far_sizes(ctx, shape, group, sizes):
    """Rows and weights whose products, or whose scales, come near the ends of fp32's range, beside ordinary rows and
    a group of zeros.  Same bars as above: nothing here is a denormal, but for elements far below their scale."""
    rows, cols, _ = shape
    x, w = make(*shape, torch.float32, 3 + sum(shape))
    x[::2] *= sizes[0]
    w *= sizes[1]
    if cols > 256:
        x[1, 128:256] = 0.0
    groups = -(-cols // group) if group else 1
    q = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((rows, groups), device="cuda")
    ctx.rmsnorm_e4m3(x, w, q, scales, 2.0 ** -120, group=group)
    ctx.sync()
    h = x.double()
    want = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + 2.0 ** -120) * w.double()
    width = group or cols
    top = torch.stack([want[:, i * width:(i + 1) * width].abs().amax(dim=1) for i in range(groups)], dim=1)
    close(scales, top / 448.0, top / 448.0 * FP32 + 2.0 ** -126, "scales")
    s = scales.double().repeat_interleave(width, dim=1)[:, :cols]
    close(q.float().double() * s, want, torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -12), "q * scale")


def backward64(dy, h, w, dres):
    h, dy = h.double(), dy.double()
    _, r = norm64(h, w)
    wdy, xhat = w.double() * dy, h * r
    dx = r * (wdy - xhat * (wdy * xhat).mean(dim=1, keepdim=True))
    size = r * (wdy.abs() + xhat.abs() * (wdy * xhat).abs().mean(dim=1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
        size = size + dres.double().abs()
    return dx, size, (dy * xhat).sum(dim=0), (dy * xhat).abs().sum(dim=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + [(9000, 512, 0)])
def test_backward(ctx, shape, dtype):
    rows, cols, _ = shape
    dy, h, dres, w = make(*shape, dtype, 2 + sum(shape), 3)
    dx, dw = torch.empty_like(dy), torch.full((cols,), 7.0, device="cuda")
    ctx.rmsnorm_backward(dy, h, w, dx, dw, EPS, dresidual=dres)
    twice = dw.clone()
    alone = torch.empty_like(dy)
    ctx.rmsnorm_backward(dy, h, w, alone, None, EPS)
    ctx.rmsnorm_backward(dy, h, w, alone, twice, EPS, accumulate=True)
    ctx.sync()
    want, size, want_w, size_w = backward64(dy, h, w, dres)
    close(dx, want, size * FP32 + want.abs() * HALF[dtype], "dx")
    # a team adds at most rows / 148 products in a row, the join 32 and 32 more: under 2^-16 for these rows
    close(dw, want_w, size_w * 2.0 ** -16, "dweight")
    want, size, _, _ = backward64(dy, h, w, None)
    close(alone, want, size * FP32 + want.abs() * HALF[dtype], "dx without dresidual")
    close(twice, 2 * want_w, size_w * 2.0 ** -15, "dweight, accumulated")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(131, 8), (20003, 40), (20001, 64), (20002, 128), (19999, 136), (5000, 256), (7, 264), (33, 896), (3000, 1536),
                                   (6, 2560), (400, 5120), (2, 7000), (1, 64)])
def test_backward_on_the_vectors_grid(ctx, shape, dtype):
    """Parts of warps and blocks of every size, more rows than teams; eps 0 and rows behind the last."""
    rows, cols = shape
    dy, h, dres, w = make(rows, cols, 0, dtype, 4 + rows + cols, 3)
    room = torch.full((rows + 2, cols), 7.0, dtype=dtype, device="cuda")
    dw = torch.empty(cols, device="cuda")
    ctx.rmsnorm_backward(dy, h, w, room[:rows], dw, 0.0, dresidual=dres)
    ctx.sync()
    d, x, wd = dy.double(), h.double(), w.double()
    r = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True))
    xhat, wdy = x * r, wd * d
    want = r * (wdy - xhat * (wdy * xhat).mean(dim=1, keepdim=True)) + dres.double()
    size = r * (wdy.abs() + xhat.abs() * (wdy * xhat).abs().mean(dim=1, keepdim=True)) + dres.double().abs()
    close(room[:rows], want, size * FP32 + want.abs() * HALF[dtype], "dx")
    # as above: a team adds at most rows / 148 products one after the other
    close(dw, (d * xhat).sum(dim=0), (d * xhat).abs().sum(dim=0) * 2.0 ** -16, "dweight")
    assert bool((room[rows:] == 7.0).all())


def test_gradient_against_differences(ctx):
    """Central differences of the fp32 forward pass: c(x) = sum(dy * y(x)) along a random direction.  With steps
    of 2^-5 the third-order term and the sums' rounding (2^-18 of 4096 terms of size ~1) stay under 2 % of a
    derivative of order sqrt(4096)."""
    x, w = make(16, 256, 0, torch.float32, 5)
    g = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.randn(x.shape, generator=g, device="cuda")
    u = torch.randn(x.shape, generator=g, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ctx.rmsnorm_backward(dy, x, w, dx, dw, EPS)

    def c(x, w):
        y = torch.empty_like(x)
        ctx.rmsnorm(x, w, y, EPS)
        return float((y.double() * dy.double()).sum())

    step = 2.0 ** -5
    along = float((dx.double() * u.double()).sum())
    assert abs((c(x + step * u, w) - c(x - step * u, w)) / (2 * step) - along) <= 0.02 * 64
    uw = torch.randn(w.shape, generator=g, device="cuda")
    along = float((dw.double() * uw.double()).sum())     # y is linear in w
    assert abs((c(x, w + step * uw) - c(x, w - step * uw)) / (2 * step) - along) <= 0.02 * 64


@pytest.mark.parametrize("cols", [4096, 1021, 20001])
@pytest.mark.parametrize("dtype", TYPES)
def test_outputs_on_their_inputs(ctx, cols, dtype):
    x, res, dy, w = make(37, cols, 0, dtype, 7, 3)
    y, h, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    dw, dw2 = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    ctx.rmsnorm(x, w, y, EPS, residual=res, residual_out=h)
    ctx.rmsnorm_backward(dy, h, w, dx, dw, EPS, dresidual=res)
    x2, res2 = x.clone(), res.clone()
    ctx.rmsnorm(x2, w, x2, EPS, residual=res2, residual_out=res2)
    assert torch.equal(x2, y) and torch.equal(res2, h)
    for at in range(3):
        ops = [dy.clone(), h.clone(), res.clone()]
        ctx.rmsnorm_backward(ops[0], ops[1], w, ops[at], dw2, EPS, dresidual=ops[2])
        assert torch.equal(ops[at], dx) and torch.equal(dw, dw2)


def test_rows_of_zeros_infinities_and_nan(ctx):
    x = torch.randn((5, 1000), device="cuda")
    x[1] = 0.0
    x[2, 3] = float("inf")
    x[3, 4] = float("nan")
    w = torch.ones(1000, device="cuda")
    y = torch.empty_like(x)
    ctx.rmsnorm(x, w, y, EPS)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((5, 8), device="cuda")
    ctx.rmsnorm_e4m3(x, w, q, scales, EPS, group=128)
    ctx.sync()
    assert bool((y[1] == 0).all()) and bool((q[1].float() == 0).all()) and bool((scales[1] == 2.0 ** -126).all())
    assert bool(y[2, 3].isnan()) and bool((y[2, 4:] == 0).all())      # inf * 0, finite * 0
    assert bool(q[2].float()[3].isnan()) and bool(y[3].isnan().all()) and bool(q[3].float().isnan().all())
    for row in (0, 4):                                                # neighbours are untouched by it
        want, _ = norm64(x[row:row + 1].double(), w)
        close(y[row:row + 1], want, want.abs() * FP32 + 1e-30)


def test_rows_further_apart_than_32_bits(ctx):
    ld, cols = (1 << 31) + 8, 512
    base = torch.empty(ld + cols, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, cols), (ld, 1))
    x.copy_(torch.randn((2, cols), device="cuda"))
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    y = torch.empty((2, cols), dtype=torch.bfloat16, device="cuda")
    ctx.rmsnorm(x, w, y, EPS)
    want, _ = norm64(x.double(), w)
    ctx.rmsnorm(x, w, x, EPS)
    ctx.sync()
    close(y, want, want.abs() * (FP32 + HALF[torch.bfloat16]) + 1e-30)
    assert torch.equal(x, y)


def test_same_bits_again_on_another_stream_and_in_a_graph(ctx):
    dy, h, dres, w = make(700, 1024, 0, torch.bfloat16, 11, 3)
    runs = []
    for stream in (None, torch.cuda.Stream()):
        dx, dw = torch.empty_like(dy), torch.empty(1024, device="cuda")
        torch.cuda.synchronize()
        ctx.rmsnorm_backward(dy, h, w, dx, dw, EPS, dresidual=dres, stream=stream)
        torch.cuda.synchronize()
        runs.append((dx, dw))
    dx, dw = torch.zeros_like(dy), torch.zeros(1024, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.rmsnorm_backward(dy, h, w, dx, dw, EPS, dresidual=dres, stream=torch.cuda.current_stream())
    # a larger call in between grows the scratch that the graph holds the address of: it stays valid
    big_dy, big_h, big_w = make(30000, 8192, 0, torch.bfloat16, 12, 2)
    ctx.rmsnorm_backward(big_dy, big_h, big_w, torch.empty_like(big_dy), torch.empty(8192, device="cuda"), EPS)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    runs.append((dx, dw))
    for other in runs[1:]:
        assert torch.equal(runs[0][0], other[0]) and torch.equal(runs[0][1], other[1])


def test_empty_and_refused(ctx):
    from gern_b200 import api
    w = torch.ones(8, device="cuda")
    dw = torch.full((8,), 3.0, device="cuda")
    none = torch.empty((0, 8), device="cuda")
    ctx.rmsnorm(none, w, none, EPS)
    ctx.rmsnorm_backward(none, none, w, none, dw, EPS, accumulate=True)
    assert bool((dw == 3.0).all())
    ctx.rmsnorm_backward(none, none, w, none, dw, EPS)
    ctx.sync()
    assert bool((dw == 0.0).all())
    x = torch.randn((4, 8), device="cuda")
    keep = x.clone()
    with pytest.raises(api.GernB200Error) as e:       # y one row below x
        ctx.rmsnorm(x[:3], w, x[1:], EPS)
    assert e.value.code == -1
    with pytest.raises(api.GernB200Error):
        ctx.rmsnorm(x, w, torch.empty_like(x), -1.0)
    with pytest.raises(api.GernB200Error) as e:
        ctx.rmsnorm_e4m3(x, w, torch.empty((4, 8), dtype=torch.uint8, device="cuda"), torch.empty((4, 1), device="cuda"),
                         EPS, group=48)
    assert e.value.code == -3
    with pytest.raises(api.GernB200Error):            # a broadcast row has no leading dimension of its own
        ctx.rmsnorm(x[:1].expand(4, 8), w, torch.empty_like(x), EPS)
    assert torch.equal(x, keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,pad,group", [(500, 3, 32), (1021, 0, 64), (509, 0, 128), (33, 0, 32)])
def test_e4m3_of_many_rows_of_one_warp_off_the_grid(ctx, cols, pad, group, dtype):
    """A warp per row whose groups' maxima meet in shared memory: enough rows that warps of many blocks run at once."""
    rows = 20001
    x, w = make(rows, cols, pad, dtype, 31 + cols)
    groups = -(-cols // group)
    q = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((rows, groups), device="cuda")
    ctx.rmsnorm_e4m3(x, w, q, scales, EPS, group=group)
    ctx.sync()
    want, _ = norm64(x.double(), w)
    top = torch.stack([want[:, i * group:(i + 1) * group].abs().amax(dim=1) for i in range(groups)], dim=1)
    close(scales, top / 448.0, top / 448.0 * FP32 + 2.0 ** -126, "scales")
    s = scales.double().repeat_interleave(group, dim=1)[:, :cols]
    close(q.float().double() * s, want, torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -12), "q * scale")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("cols", [64, 200, 510, 1021, 4096, 8192, 16384, 16400])
def test_e4m3_scale_is_the_rounded_quotient(ctx, cols, group, dtype):
    """Rows of 1 and -1 with eps 0: r is 1 and y the weight, so each scale is max |weight| / 448 rounded once, in rows of
    every width alike."""
    g = torch.Generator(device="cuda").manual_seed(41 + cols)
    x = (2.0 * torch.randint(0, 2, (5, cols), generator=g, device="cuda") - 1.0).to(dtype)
    w = (1.0 + torch.rand(cols, generator=g, device="cuda")).to(dtype)
    groups = -(-cols // group) if group else 1
    q = torch.empty((5, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((5, groups), device="cuda")
    ctx.rmsnorm_e4m3(x, w, q, scales, 0.0, group=group)
    ctx.sync()
    width = group or cols
    top = torch.stack([w[i * width:(i + 1) * width].float().amax() for i in range(groups)])
    # (in 64 bits and then rounded: 53 bits are enough for a quotient of 24-bit numbers to be rounded once)
    assert torch.equal(scales, (top.double() / 448.0).float().expand(5, groups))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 1021, 4096, 16384, 20001])
def test_operands_that_are_columns_of_one_buffer(ctx, cols, dtype):
    """Operands of one pitch side by side share no byte: the same results as from buffers of their own, and the columns
    between them left."""
    rows, gap = 9, 3
    pitch = 4 * cols + gap
    x, res, dy, w = make(rows, cols, 0, dtype, 51 + cols, 3)
    y, h, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    dw, dw2 = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    ctx.rmsnorm(x, w, y, EPS, residual=res, residual_out=h)
    ctx.rmsnorm_backward(dy, h, w, dx, dw, EPS, dresidual=res)
    room = torch.full((rows, pitch), 7.0, dtype=dtype, device="cuda")
    a, b, c, d = (room[:, i * cols:(i + 1) * cols] for i in range(4))
    a.copy_(x)
    c.copy_(res)
    ctx.rmsnorm(a, w, b, EPS, residual=c, residual_out=d)
    ctx.sync()
    close(b, y.double(), y.double().abs() * (2 * HALF[dtype] + 2 * FP32) + 1e-30, "y")
    assert torch.equal(d, h) and torch.equal(a, x) and torch.equal(c, res) and bool((room[:, 4 * cols:] == 7.0).all())
    a.copy_(dy)
    ctx.rmsnorm_backward(a, d, w, b, dw2, EPS, dresidual=c)
    ctx.sync()
    want, size, want_w, size_w = backward64(dy, h, w, res)
    close(b, want, size * FP32 + want.abs() * HALF[dtype], "dx")
    close(dw2, want_w, size_w * 2.0 ** -16, "dweight")
    assert torch.equal(a, dy) and torch.equal(d, h) and torch.equal(c, res) and bool((room[:, 4 * cols:] == 7.0).all())
    # a weight in the gap between two rows, and e4m3 bytes beside their rows
    wide = torch.full((rows, 4 * cols), 7.0, dtype=dtype, device="cuda")
    wide[:, :cols].copy_(x)
    wide[0, cols:2 * cols] = w
    bytes_ = wide.view(torch.uint8)
    q = bytes_[:, 2 * cols * x.element_size():2 * cols * x.element_size() + cols]
    scales, q2, scales2 = torch.empty((rows, 1), device="cuda"), torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty((rows, 1), device="cuda")
    ctx.rmsnorm_e4m3(wide[:, :cols], wide[0, cols:2 * cols], q, scales, EPS)
    ctx.rmsnorm_e4m3(x, w, q2, scales2, EPS)
    ctx.sync()
    want, _ = norm64(x.double(), w)
    for b8, s in ((q, scales), (q2, scales2)):
        value = b8.contiguous().view(torch.float8_e4m3fn).float().double() * s.double()
        close(value, want, torch.maximum(want.abs() * 2.0 ** -4, s.double() * 2.0 ** -10) * (1 + 2.0 ** -12), "q * scale")
    assert bool((wide[:, 3 * cols:] == 7.0).all()) and torch.equal(wide[:, :cols], x)
