"""The input stage where its arithmetic or its arguments reach an end: 8-bit scales of the smallest magnitudes,
outputs that share memory with inputs, the modules' rules, the largest batches."""
import pytest
import torch
from torch.autograd import forward_ad

from hades_amd import dist_emb, functional, ops

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -149      # float32's smallest number


def check_8bit(q, scales, steps, group):
    """q and scales of rows whose values are `steps` (whole numbers, float64 [rows, cols]) times STEP.

    A scale is top / 448 rounded to a whole number of steps: off by half a step (and by 2^-20 of one, as the quotient
    by 448 is a product corrected once).  A value in units of its scale is rounded by at most 2^-4 of itself or 2^-10,
    half the type's smallest step; one above 448 becomes 448, which loses at most 448 half steps.  A scale of 0
    (largest magnitudes of up to 224 steps) loses the value, at most 224 steps."""
    assert bool(torch.isfinite(q.float()).all()), "%d values are not finite" % int((~torch.isfinite(q.float())).sum())
    rows, cols = steps.shape
    width = group or cols
    top = steps.abs().reshape(rows, cols // width, width).amax(2)
    got = scales.cpu().double() / STEP
    assert bool(((got - top / 448).abs() <= 0.5 * (1 + 2.0 ** -20)).all())
    unit = torch.repeat_interleave(got, width, 1)
    value = q.cpu().float().double() * unit
    bound = 448 * 0.5 * (1 + 2.0 ** -20) + steps.abs() * 2.0 ** -4 + unit * 2.0 ** -10
    assert bool(((value - steps).abs() <= bound).all())


def steps_of(tops, width):
    """Groups of `width` whole numbers, the largest magnitude of each first (and last, negative)."""
    parts = torch.arange(width, dtype=torch.float64) / width
    s = (tops.double()[:, None] * parts).floor()
    s[:, 0], s[:, -1] = tops, -tops
    return s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [8, 64])
def test_8bit_groups_of_the_smallest_magnitudes(cuda_device, dtype, group):
    # every largest magnitude from 1 to 8 192 steps: scales of 0 to 18 steps.  Rows of ones normalise to 1 - 5e-7,
    # and a weight of up to 8 192 steps times that rounds to itself
    for first in range(0, 8192, 1024):
        tops = torch.arange(first + 1, first + 1025)
        steps = steps_of(tops, group).reshape(1, -1)
        x = torch.ones((2, steps.size(1)), dtype=dtype, device="cuda")
        q, scales, _ = ops.rms_norm_8bit(x, (steps[0] * STEP).float().cuda(), group=group)
        check_8bit(q, scales, steps.expand(2, -1), group)


@pytest.mark.parametrize("cols", [8, 64, 500, 4104, 16416])
@pytest.mark.parametrize("top", [1, 224, 225, 448, 464, 671, 672, 673, 1119, 448 * 13 + 223, 448 * 14 + 223])
def test_8bit_rows_of_the_smallest_magnitudes(cuda_device, cols, top):
    steps = steps_of(torch.tensor([top]), cols)
    x = torch.ones((3, cols), device="cuda")
    q, scales, _ = ops.rms_norm_8bit(x, (steps[0] * STEP).float().cuda())
    check_8bit(q, scales, steps.expand(3, -1), 0)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(cuda_device, grad):
    """A tangent never gets lost: with gradients on or off, autograd refuses a tensor that carries one."""
    t = torch.ones((4, 8), device="cuda")
    w = torch.ones(8, device="cuda")
    ids = torch.arange(4, device="cuda")
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        x, g = forward_ad.make_dual(t, t), forward_ad.make_dual(w, w)
        for call in (lambda: functional.embed(x, ids), lambda: functional.dropout(x, 0.5, 1, 0),
                     lambda: functional.dropout(t, 0.5, 1, 0, residual=x), lambda: functional.rms_norm(x, w),
                     lambda: functional.rms_norm(t, g), lambda: functional.rms_norm(t, w, residual=x),
                     lambda: functional.rms_norm(t, residual=x, dropout=(0.5, 1, 0))):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        # and one that carries none is served inside the level as outside
        assert torch.equal(functional.embed(t, ids), t) and torch.equal(functional.dropout(t, 1.0, 1, 0, residual=t), t)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("which", ["x", "residual", "view of x"])
@pytest.mark.parametrize("cols", [8, 333, 4096, 9000, 16500])      # every form of the kernel
def test_norm_in_place(cuda_device, cols, which, eight):
    """h_out may be x or the residual: h lands there, and everything is what separate outputs give."""
    g = torch.Generator().manual_seed(cols)
    x, res = (torch.randn((5, cols), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    w = torch.randn(cols, generator=g).cuda()

    def call(x, res, drop, **kw):
        if eight:
            q, scales, h = ops.rms_norm_8bit(x, w, residual=res, group=64, dropout=drop, **kw)
            return q.view(torch.uint8), scales, h
        return ops.rms_norm(x, w, residual=res, dropout=drop, **kw)
    for residual, drop in ((res, None), (res, (0.3, 1, 2)), (None, (0.3, 1, 2)), (None, None)):
        if which == "residual" and residual is None:
            continue
        want = call(x, residual, drop)
        mine, theirs = x.clone(), None if residual is None else residual.clone()
        into = theirs if which == "residual" else (mine if which == "x" else mine.view(5, cols))
        got = call(mine, theirs, drop, h_out=into)
        h = got[1] if not eight else got[2]
        assert h is into
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(theirs if which == "residual" else mine, want[1] if not eight else want[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [False, True])
def test_float32_residual_in_training_and_evaluation(cuda_device, dtype, norm):
    """16-bit rows onto a float32 stream: one rule whatever the mode, and gradients of both."""
    n, dim, drop = 70, 40, (0.25, 9, 3)
    g = torch.Generator().manual_seed(1)
    x, res = torch.randn((n, dim), generator=g).to(dtype).cuda(), torch.randn((n, dim), generator=g).cuda()
    c = torch.randn((n, dim), generator=g).cuda()
    stage = dist_emb.InputStage(dim, dtype, dropout=drop[0], norm=norm, seed=drop[1])
    x.requires_grad_(), res.requires_grad_()
    h = stage(x, res, offset=drop[2])
    h = h[1] if norm else h
    h.backward(c)
    masked = ops.dropout(x.detach().float(), *drop)
    assert h.dtype == torch.float32 and torch.equal(h, masked + res)     # the sum's one rounding, in either order
    assert torch.equal(res.grad, c)
    assert x.grad.dtype == dtype and torch.equal(x.grad, ops.dropout_grad(c, *drop).to(dtype))
    with torch.no_grad():
        again = stage(x, res, offset=drop[2])
        assert torch.equal(again[1] if norm else again, h)
        stage.eval()
        plain = stage(x, res)
        assert torch.equal(plain[1] if norm else plain, x.float() + res)


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("norm", [False, True])
def test_residuals_that_no_mode_takes(cuda_device, training, p, norm):
    stage = dist_emb.InputStage(8, torch.float32, dropout=p, norm=norm, seed=1).train(training)
    x = torch.ones((4, 8), device="cuda")
    for bad in (x[:1], x[0], x.bfloat16(), x.double(), torch.ones((2, 4, 8), device="cuda")):
        with pytest.raises(RuntimeError, match="residual must have"):
            stage(x, bad)
    with pytest.raises(RuntimeError, match="residual must have"):
        stage(x.bfloat16(), x.half())
    assert stage(x, x) is not None


def test_layers_without_seeds_draw_different_masks(cuda_device):
    """A model of default modules: no two of its layers drop the same values, in any step."""
    layers = [dist_emb.InputStage(512, torch.float32, dropout=0.5) for _ in range(3)]
    table = dist_emb.TokenEmb(64, 512, torch.float32, dropout=0.5, weight=torch.ones(64, 512))
    ids, x = torch.arange(64, device="cuda"), torch.ones((64, 512), device="cuda")
    masks = []
    for _ in range(2):
        masks += [layer(x) != 0 for layer in layers] + [table(ids) != 0]
    for i, a in enumerate(masks):
        for b in masks[:i]:
            # independent halves agree in half of 32 768 places, five standard deviations are 453
            assert abs(int((a == b).sum()) - 16384) < 453


def test_captures_of_one_leaf_on_two_streams(cuda_device):
    """Beside a graph that was captured on another stream the refusal says so; on the same stream it is served."""
    w = torch.arange(32.0, device="cuda").reshape(4, 8).requires_grad_()
    ids = torch.tensor([3, 1], device="cuda")
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0], stream=first):
        a = functional.embed(w, ids)
    with pytest.raises(RuntimeError, match="captured on another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=second):
            functional.embed(w, ids)
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[1], stream=first):
        b = functional.embed(w, ids, 2.0)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, w.detach()[ids]) and torch.equal(b, 2 * w.detach()[ids])


def test_embed_grad_of_more_than_2_to_29_positions(cuda_device):
    """A batch past 2^29 positions, whole numbers: every partial sum stays below 2^24, so the result has to be equal."""
    n, vocab, dim = (1 << 29) + 37, 1009, 8
    ids = torch.arange(n, dtype=torch.int32, device="cuda") % vocab
    ids[-5:] = -1
    rows = torch.arange(8, device="cuda")[:, None] + torch.arange(dim, device="cuda") - 7     # -7 .. 7, by position % 8
    grad = rows.to(torch.bfloat16).repeat((n + 7) // 8, 1)[:n]
    got = ops.embed_grad(grad, ids, vocab, out_dtype=torch.float32)
    # the positions of token v: v, v + vocab, ...: eight in a row (vocab is odd) meet each remainder once
    count = torch.zeros((vocab, 8), dtype=torch.int64, device="cuda")
    for first in range(0, n, 1 << 26):
        last = min(first + (1 << 26), n)
        part = ids[first:last].long()
        key = part * 8 + torch.arange(first, last, device="cuda") % 8
        count += torch.bincount(key[part >= 0], minlength=8 * vocab).view(vocab, 8)
    want = count.double() @ rows.double()
    assert float(count.sum()) == n - 5 and float(want.abs().max()) < 2 ** 24
    assert torch.equal(got.double(), want)
