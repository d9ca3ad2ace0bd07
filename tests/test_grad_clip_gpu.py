"""Global gradient norm and clipping over lists of tensors against 64-bit forms.

Bars: sums are fp64 from groups of 16 squares added in fp32 (16 additions and a product: 17 * 2^-24 of the sum,
half of that on the norm, which is then rounded once): under 2^-20 relative.  A scaled element is the product with
a coefficient that is a quotient of fp32 values: 2^-19 relative, plus half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

NORM = 2.0 ** -20
SCALED = {torch.float32: 2.0 ** -19, torch.bfloat16: 2.0 ** -19 + 2.0 ** -8}
F, B = torch.float32, torch.bfloat16


def make(sizes, dtypes, seed, offset=0):
    """Tensors one after the other in one buffer per type: odd sizes leave odd alignments."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bufs = {t: torch.randn(sum(sizes) + offset + 1, generator=g, device="cuda").to(t) for t in set(dtypes)}
    out, at = [], offset
    for n, t in zip(sizes, dtypes):
        out.append(bufs[t][at:at + n])
        at += n
    return out


def norm64(tensors):
    return float(torch.stack([t.double().square().sum() for t in tensors]).sum().sqrt())


def check(tensors, before, norm, max_norm):
    want = norm64(before)
    assert abs(float(norm) - want) <= NORM * want
    c = max_norm / want if want > max_norm else 1.0
    for got, b in zip(tensors, before):
        off = (got.double() - b.double() * c).abs()
        assert bool((off <= b.double().abs() * c * SCALED[got.dtype]).all())


LISTS = [([1], [F], 0), ([5, 0, 17], [B, F, B], 1), ([4096, 4097, 3], [F] * 3, 0), ([100003, 7, 65536], [B] * 3, 3),
         ([70000, 1, 70000], [F, B, F], 1), ([513] * 99 + [9], [B, F] * 50, 2), ([300] * 1001, [B] * 1001, 0),
         ([31, 1000] * 1250, [F, B] * 1250, 1)]


@pytest.mark.parametrize("sizes,dtypes,offset", LISTS)
def test_clip_in_place_and_apart(ctx, sizes, dtypes, offset):
    grads = make(sizes, dtypes, len(sizes), offset)
    before = [t.clone() for t in grads]
    norm = torch.empty(1, device="cuda")
    max_norm = 0.3 * norm64(before)
    for out_types in (dtypes, [F] * len(sizes)):
        outs = make(sizes, out_types, 99, (offset + 1) % 4)
        ctx.grad_clip(grads, max_norm, norm, outs=outs)
        ctx.sync()
        check(outs, before, norm, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    ctx.grad_clip(grads, max_norm, norm)
    ctx.sync()
    check(grads, before, norm, max_norm)


def test_small_norm_leaves_the_gradients_bits(ctx):
    grads = make([1000, 33], [B, F], 3)
    before = [t.clone() for t in grads]
    outs = [torch.empty_like(t) for t in grads]
    norm = torch.empty(1, device="cuda")
    big = 10.0 * norm64(before)
    ctx.grad_clip(grads, big, norm, outs=outs)
    ctx.grad_clip(grads, big, norm)
    ctx.grad_clip(grads, float("inf"), norm)
    ctx.sync()
    for t, o, b in zip(grads, outs, before):
        assert torch.equal(t, b) and torch.equal(o, b)
    ctx.grad_clip(grads, 0.0, norm)
    ctx.sync()
    assert all(bool((t == 0).all()) for t in grads)


@pytest.mark.parametrize("size,dtype", [(1e25, F), (1e25, B), (1e-30, F), (1e-30, B), (3e-42, F)])
def test_squares_beyond_fp32(ctx, size, dtype):
    """Gradients whose squares over- or underflow in fp32 still have a norm."""
    grads = [(torch.randn(5003, device="cuda") * size).to(dtype), torch.zeros(100, dtype=dtype, device="cuda")]
    norm = torch.empty(1, device="cuda")
    ctx.grad_norm(grads, norm)
    ctx.sync()
    want = norm64(grads)
    assert abs(float(norm) - want) <= NORM * want + 2.0 ** -149


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_scales_nothing(ctx, bad):
    grads = make([5000, 77], [F, B], 4)
    grads[0][4321] = bad
    before = [t.clone() for t in grads]
    norm = torch.empty(1, device="cuda")
    ctx.grad_clip(grads, 1.0, norm)
    ctx.sync()
    assert not bool(torch.isfinite(norm).any())
    for t, b in zip(grads, before):
        assert torch.equal(t.view(torch.int16 if t.dtype == B else torch.int32), b.view(torch.int16 if b.dtype == B else torch.int32))


def test_norm_then_scale_with_a_norm_from_elsewhere(ctx):
    grads = make([4000, 4000], [B, B], 5)
    before = [t.clone() for t in grads]
    norm = torch.empty(1, device="cuda")
    ctx.grad_norm(grads, norm)
    whole = norm * 2.0          # as if three other devices held as much
    ctx.grad_scale(grads, 1.0, whole)
    ctx.sync()
    for t, b in zip(grads, before):
        want = b.double() / float(whole)
        assert bool(((t.double() - want).abs() <= want.abs() * SCALED[B]).all())


def test_same_bits_again_on_another_stream_and_in_a_graph(ctx):
    grads = make([123457, 999, 40000], [B, F, B], 6)
    runs = []
    for stream in (None, torch.cuda.Stream()):
        norm, outs = torch.empty(1, device="cuda"), [torch.empty_like(t) for t in grads]
        torch.cuda.synchronize()
        ctx.grad_clip(grads, 1.0, norm, outs=outs, stream=stream)
        torch.cuda.synchronize()
        runs.append([norm] + outs)
    norm, outs = torch.zeros(1, device="cuda"), [torch.zeros_like(t) for t in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.grad_clip(grads, 1.0, norm, outs=outs, stream=torch.cuda.current_stream())
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    runs.append([norm] + outs)
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_lists_that_are_refused(ctx):
    from gern_b200 import api
    t = torch.ones(100, device="cuda")
    norm = torch.empty(1, device="cuda")
    for grads, outs in (([t, t], None), ([t[:60], t[50:]], None), ([t], [t.view(B)[100:200].view(F)]),
                        ([t[:50], t[50:]], [t[50:], t[:50]]), ([t[:50]], [t[1:51]])):
        if outs is not None and outs[0].numel() != grads[0].numel():
            continue
        with pytest.raises(api.GernB200Error) as e:
            ctx.grad_clip(grads, 1.0, norm, outs=outs)
        assert e.value.code == -1 and "overlaps" in str(e.value)
    with pytest.raises(api.GernB200Error):
        ctx.grad_clip([t], 1.0, t[:1])
    ctx.grad_norm([t, t], norm)          # reading twice is no clash: it counts twice
    ctx.sync()
    assert abs(float(norm) - 200.0 ** 0.5) <= NORM * 15
    assert bool((t == 1.0).all())
    ctx.grad_clip([], 1.0, norm)
    ctx.sync()
    assert float(norm) == 0.0


def test_a_result_inside_its_gradient_is_refused(ctx):
    """The result starts inside the gradient, reached through a view of another type."""
    from gern_b200 import api
    t, norm = torch.ones(100, device="cuda"), torch.empty(1, device="cuda")
    out = t.view(B)[50:150].view(F)
    assert out.numel() == 50 and out.data_ptr() == t.data_ptr() + 100
    with pytest.raises(api.GernB200Error) as e:
        ctx.grad_clip([t[:50]], 1.0, norm, outs=[out])
    assert e.value.code == -1 and "overlaps" in str(e.value)
    ctx.sync()
    assert bool((t == 1.0).all())
