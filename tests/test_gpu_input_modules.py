"""The input stage as a model uses it: the differentiable functions, TokenEmb, and DistEmb with dropout and
norm, eagerly and captured, against the definitions in 64 bits and the operators' own calls."""
import numpy as np
import pytest
import torch

from hades_amd import dist_emb, functional, ops
from test_gpu_input_stage import U, factors, rows_of, token_ids, within

pytestmark = pytest.mark.gpu


def test_functions_together_against_64_bit_autograd(cuda_device):
    """Two layers of an input stage - lookup, dropout, norm with residual - and their gradients against torch's
    autograd over the same formulas in 64 bits on the CPU, masks included."""
    n, vocab, dim, scale, eps = 200, 60, 96, 9.8, 1e-5
    d1, d2, d3 = (0.1, 1, 0), (0.2, 1, 1), (0.3, 1, 2)
    ids = token_ids(n, vocab, 1, 0.1)
    w = [rows_of((vocab, dim), torch.float32, 2, 0.1), rows_of((dim,), torch.float32, 3) + 1,
         rows_of((dim,), torch.float32, 4) + 1, rows_of((n, dim), torch.float32, 5)]
    cy, ch = rows_of((n, dim), torch.float32, 6), rows_of((n, dim), torch.float32, 7)

    leaves = [t.cuda().requires_grad_() for t in w]
    table, g1, g2, res = leaves
    x = functional.embed(table, ids.cuda(), scale, padding_idx=3, dropout=d1)
    y, h = functional.rms_norm(x, g1, eps, residual=res, dropout=d2)
    z = functional.dropout(y, *d3, residual=h)
    y2, h2 = functional.rms_norm(z, g2, eps)
    assert h2 is z
    out = [y2, h2]
    torch.autograd.backward(out, [cy.cuda(), ch.cuda()])

    dl = [t.double().requires_grad_() for t in w]
    dt, dg1, dg2, dres = dl
    live = (ids >= 0)[:, None]
    rows = torch.where((ids == 3)[:, None], dt.detach()[ids.clamp(min=0)], dt[ids.clamp(min=0)]) * live

    def norm(v, g):
        return v * torch.rsqrt(v.square().mean(1, keepdim=True) + eps) * g
    xd = rows * scale * factors(n, dim, d1)
    hd = dres + xd * factors(n, dim, d2)
    zd = norm(hd, dg1) * factors(n, dim, d3) + hd
    outd = [norm(zd, dg2), zd]
    torch.autograd.backward(outd, [cy.double(), ch.double()])
    # every value passes through fewer than 40 float32 operations and sums of fewer than 400 terms whose partial
    # results are at most a few hundred times the largest result's magnitude divided by the sums' length
    for got, want in list(zip(out, outd)) + [(a.grad, b.grad) for a, b in zip(leaves, dl)]:
        within(got.detach(), want.detach(), 400 * U * float(want.detach().abs().max()))
    assert not table.grad[3].any()


def test_gradients_against_differences(cuda_device):
    """functional.embed and functional.dropout are linear: a difference of any size gives the gradient."""
    ids = torch.tensor([2, 0, 2, -1, 5], device="cuda")
    w = rows_of((6, 9), torch.float32, 1).cuda().requires_grad_()
    c = rows_of((5, 9), torch.float32, 2).cuda()
    drop = (0.4, 8, 3)
    y = functional.dropout(functional.embed(w, ids, 2.0, dropout=(0.2, 8, 1)), *drop)
    y.backward(c)
    for i, j in ((2, 0), (0, 8), (5, 4), (1, 1)):
        moved = w.detach().clone()
        moved[i, j] += 1.0
        f = [functional.dropout(functional.embed(t, ids, 2.0, dropout=(0.2, 8, 1)), *drop) for t in (moved, w.detach())]
        want = float(((f[0] - f[1]).double() * c.double()).sum())
        # the difference of two float32 outputs of magnitude below 16, five terms
        assert abs(float(w.grad[i, j]) - want) <= 5 * 16 * 4 * U * float(c.abs().max()) + 1e-30


def test_only_h_or_only_y_is_used(cuda_device):
    x = rows_of((8, 40), torch.bfloat16, 1).cuda().requires_grad_()
    r = rows_of((8, 40), torch.float32, 2).cuda().requires_grad_()
    g = rows_of((40,), torch.bfloat16, 3).cuda().requires_grad_()
    c = rows_of((8, 40), torch.float32, 4).cuda()
    drop = (0.25, 3, 4)
    y, h = functional.rms_norm(x, g, residual=r, dropout=drop)
    h.backward(c)
    assert torch.equal(r.grad, c) and g.grad is None
    assert torch.equal(x.grad, ops.dropout_grad(c, *drop).bfloat16())
    x.grad = r.grad = None
    y, h = functional.rms_norm(x, g, residual=r, dropout=drop)
    y.sum().backward()                                   # an expanded gradient
    _, hh, rstd = ops.rms_norm(x.detach(), g.detach(), residual=r.detach(), dropout=drop)
    want = ops.rms_norm_grad(torch.ones_like(x), hh, g.detach(), rstd, dropout=drop)
    assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[1]) and torch.equal(g.grad, want[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", [False, True])
def test_token_emb_module(cuda_device, dtype, norm):
    vocab, dim = 300, 64
    emb = dist_emb.TokenEmb(vocab, dim, dtype, scale=8.0, padding_idx=0, dropout=0.1, norm=norm, seed=21,
                            weight=rows_of((vocab, dim), dtype, 1))
    ids = token_ids(400, vocab, 2, 0.1).view(20, 20).cuda()
    res = rows_of((20, 20, dim), dtype, 3).cuda()
    for call in range(3):                                # every call draws the next mask
        drop = (0.1, 21, call)
        emb.zero_grad()
        if norm:
            y, h = emb(ids, residual=res)
            x = ops.embed(emb.weight.detach(), ids, scale=8.0)
            wy, wh, rstd = ops.rms_norm(x, emb.stage.weight.detach(), residual=res, dropout=drop)
            assert torch.equal(y, wy) and torch.equal(h, wh)
            y.backward(res)
            gx, _, gw = ops.rms_norm_grad(res, wh, emb.stage.weight.detach(), rstd, dropout=drop)
            assert torch.equal(emb.stage.weight.grad, gw)
            want = ops.embed_grad(gx, ids, vocab, scale=8.0, padding_idx=0)
        else:
            y = emb(ids)
            assert torch.equal(y, ops.embed(emb.weight.detach(), ids, scale=8.0, dropout=drop))
            y.backward(res)
            want = ops.embed_grad(res, ids, vocab, scale=8.0, padding_idx=0, dropout=drop)
        assert torch.equal(emb.weight.grad, want)
    state = emb.state_dict()
    other = dist_emb.TokenEmb(vocab, dim, dtype, scale=8.0, padding_idx=0, dropout=0.1, norm=norm, seed=21)
    other.load_state_dict(state)
    a, b = emb(ids), other(ids)                          # a resumed run draws what the first would have drawn
    assert all(torch.equal(p, q) for p, q in zip(a if norm else [a], b if norm else [b]))
    emb.eval()
    with torch.no_grad():
        plain = emb(ids)
    x = ops.embed(emb.weight.detach(), ids, scale=8.0)
    if norm:
        assert torch.equal(plain[0], ops.rms_norm(x, emb.stage.weight.detach())[0]) and torch.equal(plain[1], x)
        q, s, h = emb.forward_8bit(ids, residual=res, group=32)
        wq, wsc, wh = ops.rms_norm_8bit(x, emb.stage.weight.detach(), residual=res, group=32)
        assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, wsc) and torch.equal(h, wh)
    else:
        assert torch.equal(plain, x)


@pytest.mark.parametrize("pin", [True, False])
def test_dist_emb_with_dropout_and_norm(cuda_device, pin):
    """DistEmb(dropout=, norm=) against the explicit calls: rows, normalised rows, and the tables after two steps
    of the sparse optimizer are bit-equal."""
    from hades_amd import sparse_optim
    N, D, n = 3000, 48, 2000
    weight = rows_of((N, D), torch.float32, 1, 0.05)
    hot = torch.arange(N) % 7
    emb = dist_emb.DistEmb(N, D, torch.float32, "emb", cache_rate=0.2, hotness_list=hot, hot_threshold=6,
                           weight=weight.clone(), pin_memory=pin, dropout=0.2, norm=True, seed=4)
    opt = dist_emb.SparseAdagrad([emb.sparse_emb], lr=0.05)
    ref = sparse_optim.SparseAdagrad(weight.clone().pin_memory() if pin else weight.clone().cuda(),
                                     emb.sparse_emb.hot_ids, lr=0.05)
    gamma = emb.stage.weight.detach()
    emb.train()
    for step in range(2):
        ids = token_ids(n, N, 10 + step).cuda()
        res = rows_of((n, D), torch.float32, 20 + step).cuda()
        c = rows_of((n, D), torch.float32, 30 + step).cuda()
        emb.stage.weight.grad = None
        y, h = emb(ids, residual=res)
        rows, state = ref.forward_keyed(ids)
        wy, wh, rstd = ops.rms_norm(rows, gamma, residual=res, dropout=(0.2, 4, step))
        assert torch.equal(y, wy) and torch.equal(h, wh)
        torch.autograd.backward([y, h], [c, c])
        gx, _, gw = ops.rms_norm_grad(c, wh, gamma, rstd, grad_h=c, dropout=(0.2, 4, step))
        assert torch.equal(emb.stage.weight.grad, gw)
        opt.step()
        ref.backward_keyed(state, gx, average="mean")
        torch.cuda.synchronize()
    for k in ("cold_w", "cold_s", "hot_w", "hot_s"):
        assert torch.equal(getattr(opt._state["emb"], k).cpu(), getattr(ref, k).cpu()), k
    emb.eval()
    ids = token_ids(100, N, 50).cuda()
    q, s, h = emb.forward_8bit(ids, group=16)
    rows = ref.fetch(ids)
    wq, wsc, _ = ops.rms_norm_8bit(rows, gamma, group=16)
    assert torch.equal(h, rows) and torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, wsc)
    assert emb.sparse_emb.trace == []
    plain = dist_emb.DistEmb(N, D, torch.float32, "plain", cache_rate=0, weight=weight.clone(), pin_memory=pin)
    assert plain.stage is None and torch.equal(plain(ids).cpu(), weight[ids.cpu()])
    with pytest.raises(RuntimeError, match="residual and offset"):
        plain(ids, residual=rows)
    with pytest.raises(RuntimeError, match="goes with norm"):
        plain.forward_8bit(ids)


def test_captured_training_step(cuda_device):
    """forward and backward of TokenEmb with norm in one graph; the graph counts its masks up itself.  Replays with
    eager work between them give the gradients of the eager step."""
    vocab, dim, n = 200, 80, 150
    emb = dist_emb.TokenEmb(vocab, dim, torch.bfloat16, scale=4.0, dropout=0.2, norm=True, seed=5)
    ids, c = token_ids(n, vocab, 1).cuda(), rows_of((n, dim), torch.bfloat16, 2).cuda()
    res = rows_of((n, dim), torch.bfloat16, 3).cuda()
    offset = torch.zeros(1, dtype=torch.int64, device="cuda")

    def eager(number):
        x = ops.embed(emb.weight.detach(), ids, scale=4.0)
        y, h, rstd = ops.rms_norm(x, emb.stage.weight.detach(), residual=res, dropout=(0.2, 5, number))
        gx, _, gw = ops.rms_norm_grad(c, h, emb.stage.weight.detach(), rstd, dropout=(0.2, 5, number))
        return y, gw, ops.embed_grad(gx, ids, vocab, scale=4.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        emb(ids, residual=res, offset=offset)[0].backward(c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    emb.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = emb(ids, residual=res, offset=offset)
        y.backward(c)
        offset.add_(1)
    for turn in range(4):
        ids.copy_(token_ids(n, vocab, 5 + turn, 0.1))
        graph.replay()
        want = eager(turn)
        torch.cuda.synchronize()
        for a, b in zip((y, emb.stage.weight.grad, emb.weight.grad), want):
            assert torch.equal(a, b)


def test_capture_beside_a_living_eager_graph_is_refused(cuda_device):
    emb = dist_emb.TokenEmb(50, 16, torch.float32, dropout=0.5)
    ids = torch.arange(20, device="cuda")
    offset = torch.zeros(1, dtype=torch.int64, device="cuda")
    alive = emb(ids)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(graph):
            emb(ids, offset=offset)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="needs an offset tensor"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            emb(ids)
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                        # gone: nothing to refuse
        out = emb(ids, offset=offset)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.embed(emb.weight.detach(), ids, dropout=(0.5, 0, 0)))


@pytest.mark.parametrize("norm", [True, False])
def test_capture_without_gradients_beside_a_living_eager_graph(cuda_device, norm):
    """A captured forward that records no graph has no backward pass to refuse: it gives what the eager call gives,
    on every replay, while the eager graph of the same leaves lives and is run backward between replays."""
    emb = dist_emb.TokenEmb(50, 16, torch.float32, dropout=0.5, norm=norm)
    ids = torch.arange(20, device="cuda")
    first = lambda out: out[0] if norm else out
    offset = torch.zeros(1, dtype=torch.int64, device="cuda")
    alive = first(emb(ids))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = first(emb(ids, offset=offset))
    assert not out.requires_grad and alive.requires_grad
    for replay in range(3):
        offset.fill_(replay)
        graph.replay()
        torch.cuda.synchronize()
        x = emb.weight.detach()
        if norm:
            want = ops.rms_norm(ops.embed(x, ids), emb.stage.weight.detach(), dropout=(0.5, 0, replay))[0]
        else:
            want = ops.embed(x, ids, dropout=(0.5, 0, replay))
        assert torch.equal(out, want)
        alive.sum().backward(retain_graph=True)
    torch.cuda.synchronize()
    assert emb.weight.grad is not None


def test_offset_tensor_changed_before_backward_is_refused(cuda_device):
    x = rows_of((4, 8), torch.float32, 1).cuda().requires_grad_()
    offset = torch.zeros(1, dtype=torch.int64, device="cuda")
    y = functional.dropout(x, 0.5, 1, offset)
    offset.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))


def test_module_refusals(cuda_device):
    with pytest.raises(RuntimeError, match="dropout must lie"):
        dist_emb.InputStage(8, torch.float32, dropout=1.5)
    with pytest.raises(RuntimeError, match="padding_idx"):
        dist_emb.TokenEmb(10, 8, torch.float32, padding_idx=10)
    with pytest.raises(RuntimeError, match="weight must be"):
        dist_emb.TokenEmb(10, 8, torch.float32, weight=torch.zeros(10, 9))
