"""The input-stage operators on the GPU against plain implementations in 64 bits: embedding with scaling and
its gradient, dropout from a counter, RMS norm with residual, 8-bit output and gradient.

Tolerances.  u = 2^-24 is half a step of float32, H(t) = torch.finfo(t).eps / 2 half a step of the stored
type.  A value computed by k float32 operations on terms whose magnitudes sum to S is off by at most about
k * u * S (each operation adds half a step of something no larger than S); storing it adds H * |value|, and
where the type's smallest normal number is reached, half of its smallest step."""
import numpy as np
import pytest
import torch

from hades_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the type's smallest step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound):
    """|got - want| <= bound, elementwise, with equal infinities and NaN."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.cpu() if isinstance(bound, torch.Tensor) else torch.full_like(want, bound)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= bound))
    assert not bad.any(), "%d of %d off, worst %.3g over its bound" % (
        int(bad.sum()), bad.numel(), float(((got - want).abs() / bound)[bad].max()))


# ---- the definitions, on the CPU --------------------------------------------------------------------
def philox(counter, key, rounds=7):
    """Philox4x32 over numpy arrays of uint64 words below 2^32."""
    low, c = np.uint64(0xFFFFFFFF), [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def kept(rows, cols, p, seed, offset):
    """bool [rows, cols]; rows a number or the row numbers"""
    rows = np.arange(rows) if np.isscalar(rows) else np.asarray(rows)
    seed &= (1 << 64) - 1
    pieces = -(-cols // 8)
    r, c = np.meshgrid(rows.astype(np.uint64), np.arange(pieces, dtype=np.uint64), indexing="ij")
    words = philox((c, r, np.full_like(c, offset & 0xFFFFFFFF), np.full_like(c, offset >> 32)),
                   (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    return torch.from_numpy(bits.reshape(len(rows), -1)[:, :cols].astype(np.int64) >= threshold(p))


def factors(rows, cols, drop):
    """What dropout multiplies with, float64 [rows, cols]."""
    if drop is None or threshold(drop[0]) == 0:
        return torch.ones((rows if np.isscalar(rows) else len(rows), cols), dtype=torch.float64)
    p, seed, offset = drop
    t = threshold(p)
    return kept(rows, cols, p, seed, int(offset)).double() * (0.0 if t == 65536 else 65536 / (65536 - t))


def rows_of(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype)


def token_ids(n, vocab, seed, padded=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * np.log(vocab + 1)).long() - 1).clamp(0, vocab - 1)
    ids = ids * 7919 % vocab
    if padded:
        ids[torch.rand(n, generator=g) < padded] = -1
    return ids


# ---- dropout ------------------------------------------------------------------------------------------
def test_generator_known_answers():
    # the published known-answer vectors of Philox4x32 for an all-zero counter and key
    assert ["%08x" % int(w) for w in philox((0, 0, 0, 0), (0, 0), 7)] == ["5f6fb709", "0d893f64", "4f121f81", "4f730a48"]
    assert ["%08x" % int(w) for w in philox((0, 0, 0, 0), (0, 0), 10)] == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 1023), (129, 64), (64, 1001), (33, 4096)])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 1.0])
def test_dropout_against_the_definition(cuda_device, dtype, rows, cols, p):
    seed, offset = -5, (7 << 32) + 11
    x, r = rows_of((rows, cols), dtype, 1), rows_of((rows, cols), dtype, 2)
    f = factors(rows, cols, (p, seed, offset))
    got = ops.dropout(x.cuda(), p, seed, offset)
    grad = ops.dropout_grad(x.cuda(), p, seed, offset)
    assert torch.equal(got, grad)
    assert torch.equal(got.cpu() != 0, (f != 0) & (x != 0))                  # the mask itself, value by value
    want = x.double() * f
    within(got, want, want.abs() * (2 * U + half_step(dtype)) + tiny(dtype))
    got = ops.dropout(x.cuda(), p, seed, offset, residual=r.cuda())
    want = x.double() * f + r.double()
    within(got, want, (3 * U) * ((x.double() * f).abs() + r.double().abs()) + half_step(dtype) * want.abs() + tiny(dtype))


def test_dropout_zeroes_what_is_not_a_number_and_counts_its_share(cuda_device):
    x = torch.full((256, 1000), float("nan"))
    x[:, ::2] = float("inf")
    keep = kept(256, 1000, 0.25, 3, 9)
    got = ops.dropout(x.cuda(), 0.25, 3, 9).cpu()
    assert bool((got[~keep] == 0).all()) and bool((~torch.isfinite(got[keep])).all())
    # 256000 draws of share 0.25: five standard deviations are 0.0043
    assert abs(float((~keep).double().mean()) - 0.25) < 0.0043
    other = kept(256, 1000, 0.25, 3, 10)
    assert abs(float((keep != other).double().mean()) - 2 * 0.25 * 0.75) < 0.006    # another offset, another mask


def test_dropout_strides_views_and_aliases(cuda_device):
    base = rows_of((40, 3, 300), torch.bfloat16, 4).cuda()
    view = base[:, 1, 5:282]                      # rows 900 apart that begin at an odd element
    assert not view.is_contiguous()
    want = ops.dropout(view.contiguous(), 0.3, 1, 2)
    assert torch.equal(ops.dropout(view, 0.3, 1, 2), want)
    wide = base[:, :, 5:282]                      # [40, 3, 277]: rows 300 apart
    assert torch.equal(ops.dropout(wide, 0.3, 1, 2), ops.dropout(wide.contiguous(), 0.3, 1, 2))
    x = base[:, 0].contiguous()
    res = base[:, 2].contiguous()
    want = ops.dropout(x, 0.3, 1, 2, residual=res)
    a, b = x.clone(), res.clone()
    assert torch.equal(ops.dropout(a, 0.3, 1, 2, residual=res, out=a), want) and torch.equal(a, want)
    assert torch.equal(ops.dropout(x, 0.3, 1, 2, residual=b, out=b), want)
    one = rows_of((7,), torch.float32, 1).cuda()
    assert torch.equal(ops.dropout(one, 0.5, 1, 2), ops.dropout(one.view(1, 7), 0.5, 1, 2).view(7))
    for shape in ((0, 8), (8, 0), (0,)):
        assert ops.dropout(torch.empty(shape, device="cuda"), 0.5, 1, 2).shape == shape


# ---- embedding ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 50, 4096), (7, 13, 8), (100, 77, 33), (513, 1000, 64),
                                         (64, 300, 1001), (2000, 90, 128)])
@pytest.mark.parametrize("scale,drop", [(1.0, None), (22.627, None), (8.0, (0.1, 5, 6))])
def test_embed_is_the_rounded_product(cuda_device, dtype, n, vocab, dim, scale, drop):
    w = rows_of((vocab, dim), dtype, 1)
    ids = token_ids(n, vocab, 2)
    ids[::5] = torch.tensor([-1, vocab, -(1 << 40), 1 << 40])[torch.arange(len(ids[::5])) % 4]
    live = (ids >= 0) & (ids < vocab)
    f32 = torch.tensor(scale, dtype=torch.float32).double()          # the scale as the kernel gets it
    factor = (f32 * factors(n, dim, drop)).float()                    # ... and its product with dropout's factor
    want = (torch.where(live[:, None], w[ids.clamp(0, vocab - 1)].float() * factor, torch.zeros(()))).to(dtype)
    got = ops.embed(w.cuda(), ids.cuda(), scale=scale, dropout=drop)
    assert got.dtype == dtype and torch.equal(got.cpu(), want)
    if bool((ids.abs() < 2 ** 31).all()):
        assert torch.equal(ops.embed(w.cuda(), ids.int().cuda(), scale=scale, dropout=drop).cpu(), want)


def test_embed_shapes_strides_and_out(cuda_device):
    big = rows_of((50, 100), torch.float16, 1).cuda()
    table = big[:, 3:80]
    ids = token_ids(60, 50, 3).view(3, 4, 5).cuda()
    got = ops.embed(table, ids)
    assert got.shape == (3, 4, 5, 77) and torch.equal(got, table[ids])
    out = torch.empty((3, 4, 5, 77), dtype=torch.float16, device="cuda")
    assert ops.embed(table, ids, out=out) is out and torch.equal(out, got)
    assert torch.equal(ops.embed(table, ids.int()[1, 2, 3]), table[ids[1, 2, 3]])   # one id, no dimension
    assert ops.embed(table, ids[:0]).shape == (0, 4, 5, 77)
    empty = ops.embed(big[:0], ids)                # a table of no rows: padding only
    assert empty.shape == (3, 4, 5, 100) and not empty.any()
    # dropout's row is the token's position: the same mask as dropout after the lookup
    x = ops.embed(table, ids)
    assert torch.equal(ops.embed(table, ids, dropout=(0.4, 1, 2)), ops.dropout(x, 0.4, 1, 2))


def want_grad(g, ids, vocab, scale, drop, padding_idx=None, base=None):
    """(gradient, bound without the stored type's part) in float64"""
    n, dim = g.shape
    f = torch.tensor(scale, dtype=torch.float32).double() * factors(n, dim, drop)
    live = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        live &= ids != padding_idx
    rows = (g.double() * f)[live]
    total = torch.zeros((vocab, dim), dtype=torch.float64).index_add_(0, ids[live], rows)
    size = torch.zeros((vocab, dim), dtype=torch.float64).index_add_(0, ids[live], rows.abs())
    count = torch.bincount(ids[live], minlength=vocab).double()[:, None]
    if base is not None:
        total, size, count = total + base.double(), size + base.double().abs(), count + 1
    return total, (count + 2) * U * size      # count products and additions, and the factor's own rounding


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None),
                                             (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 70, 64), (8, 3, 8), (31, 5, 100), (33, 1, 40), (257, 300, 64),
                                         (500, 1000, 333), (3000, 17, 128), (4097, 700, 8), (2000, 50, 1001)])
@pytest.mark.parametrize("drop,padded", [(None, 0.0), ((0.3, 11, 12), 0.3)])
def test_embed_grad_against_64_bits(cuda_device, dtype, out_dtype, n, vocab, dim, drop, padded):
    g = rows_of((n, dim), dtype, 5)
    ids = token_ids(n, vocab, 6, padded)
    want, bound = want_grad(g, ids, vocab, 3.7, drop)
    kw = dict(scale=3.7, dropout=drop, out_dtype=out_dtype)
    got = ops.embed_grad(g.cuda(), ids.cuda(), vocab, **kw)
    stored = out_dtype or dtype
    assert got.dtype == stored
    within(got, want, bound + half_step(stored) * (want.abs() + bound) + tiny(stored))
    assert torch.equal(got, ops.embed_grad(g.cuda(), ids.int().cuda(), vocab, **kw))      # and the same bits again
    absent = torch.ones(vocab, dtype=torch.bool)
    absent[ids[ids >= 0]] = False
    assert not got.cpu()[absent].any()


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                             (torch.bfloat16, torch.bfloat16)])
def test_embed_grad_accumulates_and_leaves_absent_rows(cuda_device, dtype, out_dtype):
    n, vocab, dim = 700, 400, 72
    g, ids = rows_of((n, dim), dtype, 1), token_ids(n, vocab, 2, 0.2)
    wide = rows_of((vocab, 100), out_dtype, 3)
    out = wide.cuda()[:, 10:82]                     # rows 100 apart
    want, bound = want_grad(g, ids, vocab, 2.0, None, padding_idx=int(ids.clamp(min=0).mode().values), base=wide[:, 10:82])
    got = ops.embed_grad(g.cuda(), ids.cuda(), vocab, scale=2.0, padding_idx=int(ids.clamp(min=0).mode().values), out=out,
                         accumulate=True)
    assert got is out
    within(got, want, bound + half_step(out_dtype) * (want.abs() + bound))
    absent = torch.ones(vocab, dtype=torch.bool)
    absent[ids[ids >= 0]] = False
    absent[int(ids.clamp(min=0).mode().values)] = True
    assert torch.equal(out.cpu()[absent], wide[:, 10:82][absent])
    # without accumulate the strided output is overwritten, and nothing beside it
    around = wide.cuda()
    ops.embed_grad(g.cuda(), ids.cuda(), vocab, out=around[:, 10:82])
    assert torch.equal(around[:, :10].cpu(), wide[:, :10]) and torch.equal(around[:, 82:].cpu(), wide[:, 82:])
    assert not around[:, 10:82].cpu()[absent & (torch.arange(vocab) != int(ids.clamp(min=0).mode().values))].any()


@pytest.mark.parametrize("n", [1, 7, 8, 9, 31, 32, 33, 64, 255, 1024, 9000, 70000])
def test_embed_grad_of_one_token(cuda_device, n):
    # every position holds the same token: one sum across all chunk borders; whole numbers sum exactly
    g = (torch.arange(n * 16, dtype=torch.float32) % 7).view(n, 16).cuda()
    ids = torch.full((n,), 3, dtype=torch.int64, device="cuda")
    got = ops.embed_grad(g, ids, 5)
    assert torch.equal(got[3], g.sum(0)) and not got[[0, 1, 2, 4]].any()
    none = ops.embed_grad(g, torch.full_like(ids, -1), 5)
    assert not none.any()
    assert not ops.embed_grad(g, ids, 5, padding_idx=3).any()


@pytest.mark.parametrize("vocab", [1, 255, 257, 40_000, 262_145, 600_000, 1 << 20, (1 << 20) + 1])
@pytest.mark.parametrize("n", [1, 64, 65, 1023, 1024, 1025, 131_072, 131_073])
def test_embed_grad_sorts_every_batch_in_order(cuda_device, n, vocab):
    """All forms of the sort (one tile, tiles, radix; tables on both sides of their limits).  The columns' weights
    1, k and k^2 of every position k (mod 61) are whole numbers whose sums float32 holds exactly for the
    tokens that are looked at: each token has to get its own positions, no other's and none twice."""
    ids = token_ids(n, vocab, 3, 0.1)
    ids[0] = vocab - 1
    k = torch.arange(n) % 61
    g = torch.stack((torch.ones(n), k.float(), (k * k).float()), 1)
    want = torch.zeros((vocab, 3), dtype=torch.float64).index_add_(0, ids[ids >= 0], g[ids >= 0].double())
    assert float(want.max()) < 2 ** 24 * 16      # beyond 2^24 the sum's steps may round
    got = ops.embed_grad(g.cuda(), ids.cuda(), vocab).double().cpu()
    exact = want.max(1).values < 2 ** 24
    assert torch.equal(got[exact], want[exact])
    within(got, want, want * (n * U))
    out = torch.full((vocab, 3), 0.5, device="cuda")
    got = ops.embed_grad(g.cuda(), ids.int().cuda(), vocab, out=out, accumulate=True, padding_idx=vocab - 1).double().cpu()
    want[vocab - 1] = 0
    small = want.max(1).values < 2 ** 22
    assert torch.equal(got[small], want[small] + 0.5)


@pytest.mark.parametrize("vocab", [2, 257, 40_000, 1 << 20])
@pytest.mark.parametrize("n", [2047, 2048, 2049, 3073, 4095, 4096, 4097])
def test_embed_grad_of_a_few_steps_a_wave(cuda_device, n, vocab):
    """Batches on both sides of one and two kernels.  Every sum of the columns 1 and k mod 61 is a whole number below
    2^24 (4 097 * 60 = 245 820), so float32 holds each partial sum and the result has to be equal."""
    k = torch.arange(n) % 61
    g = torch.stack((torch.ones(n), k.float()), 1)
    for kind in ("power law", "one token", "two tokens in turn", "last token"):
        ids = token_ids(n, vocab, 3, 0.1)
        if kind == "one token":
            ids.fill_(vocab // 2)
        elif kind == "two tokens in turn":
            ids = (torch.arange(n) % 2) * (vocab - 1)
        elif kind == "last token":
            ids[n // 2:] = vocab - 1
        want = torch.zeros((vocab, 2), dtype=torch.float64).index_add_(0, ids[ids >= 0], g[ids >= 0].double())
        for i in (ids, ids.int()):
            assert torch.equal(ops.embed_grad(g.cuda(), i.cuda(), vocab).double().cpu(), want), kind
    # random values: the same bits from run to run
    ids = token_ids(n, vocab, 5, 0.0)
    x = torch.randn(n, 96, generator=torch.Generator().manual_seed(n)).cuda()
    first = ops.embed_grad(x, ids.cuda(), vocab)
    assert torch.equal(first, ops.embed_grad(x, ids.cuda(), vocab))
    exact = torch.zeros((vocab, 96), dtype=torch.float64).index_add_(0, ids, x.double().cpu())
    size = torch.zeros((vocab, 96), dtype=torch.float64).index_add_(0, ids, x.double().abs().cpu())
    within(first.double().cpu(), exact, size * (n * U))


def test_embed_grad_of_no_tokens_and_strided_rows(cuda_device):
    g = rows_of((9, 4, 50), torch.bfloat16, 1).cuda()
    ids = token_ids(9, 6, 2).cuda()
    rows = g[:, 2, 3:40]
    assert torch.equal(ops.embed_grad(rows, ids, 6), ops.embed_grad(rows.contiguous(), ids, 6))
    empty = ops.embed_grad(g[:0, 0], ids[:0], 6)
    assert empty.shape == (6, 50) and not empty.any()
    assert ops.embed_grad(g[:, 0], torch.full_like(ids, -1), 0).shape == (0, 50)
    nan = g[:, 0].clone()
    nan[0] = float("nan")                          # a padded position's row is not read into a sum
    ids = torch.tensor([-1, 0, 1, 2, 3, 4, 5, 0, 1], device="cuda")
    assert torch.isfinite(ops.embed_grad(nan, ids, 6)).all()


# ---- RMS norm -------------------------------------------------------------------------------------------
def want_norm(x, w, eps, residual, drop):
    """float64 (y, h, rstd) and what h may be off by"""
    f = factors(x.shape[0], x.shape[1], drop)
    xf = x.double() * f
    h = xf if residual is None else xf + residual.double()
    off = 3 * U * (xf.abs() + (0 if residual is None else residual.double().abs()))
    rstd = 1 / torch.sqrt(h.square().mean(1) + eps)
    y = h * rstd[:, None] * (1 if w is None else w.double())
    return y, h, rstd, off


def rstd_bound(h, off, rstd):
    """Relative bound of rstd: the sum of squares (its terms positive: cols additions in the worst order, each
    half a step), what h is off by, and a handful of operations; half of it for the root."""
    ss = h.square().sum(1)
    return 0.5 * (h.shape[1] * U + 2 * (h.abs() * off).sum(1) / ss.clamp(min=1e-300)) + 8 * U


@pytest.mark.parametrize("dtype,stream,wtype", [
    (torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
    (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float16, torch.float32),
    (torch.float16, torch.float32, torch.float16)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (70, 64), (33, 100), (5, 250), (17, 512), (6, 1000), (4, 2048),
                                       (3, 4001), (2, 8192), (2, 16000), (1, 16384), (2, 16392), (1, 40001)])
@pytest.mark.parametrize("mode", ["plain", "residual", "dropout"])
def test_rms_norm_against_64_bits(cuda_device, dtype, stream, wtype, rows, cols, mode):
    x, w = rows_of((rows, cols), dtype, 1), rows_of((cols,), wtype, 2) + 1
    r = rows_of((rows, cols), stream, 3, 4.0) if mode != "plain" else None
    drop = (0.2, 1 << 63, 17) if mode == "dropout" else None
    eps = 1e-5
    y, h, rstd, off = want_norm(x, w, eps, r, drop)
    gy, gh, gr = ops.rms_norm(x.cuda(), w.cuda(), eps, residual=None if r is None else r.cuda(), dropout=drop)
    rel = rstd_bound(h, off, rstd)
    within(gr, rstd, rel * rstd)
    ybound = y.abs() * (rel[:, None] + 3 * U) + off * rstd[:, None] * w.double().abs()
    within(gy, y, ybound + half_step(dtype) * (y.abs() + ybound) + tiny(dtype))
    if mode == "plain":
        assert gh.data_ptr() and gy.dtype == dtype
    else:
        assert gh.dtype == stream
        within(gh, h, off + half_step(stream) * (h.abs() + off) + tiny(stream))


def test_rms_norm_without_weight_views_and_aliases(cuda_device):
    base = rows_of((6, 5, 700), torch.bfloat16, 1).cuda()
    view = base[:, :, 3:516]
    y, h, rstd = ops.rms_norm(view)
    assert h is view and y.shape == view.shape and rstd.shape == (6, 5)
    y2, _, _ = ops.rms_norm(view.contiguous(), torch.ones(513, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(y, y2)
    res = rows_of((6, 5, 513), torch.float32, 2).cuda()
    y, h, _ = ops.rms_norm(view, residual=res)
    again = res.clone()
    y2, h2, _ = ops.rms_norm(view, residual=again, h_out=again)          # the residual stream in place
    assert h2 is again and torch.equal(h, again) and torch.equal(y, y2)
    long = rows_of((2, 20000), torch.bfloat16, 3).cuda()
    res = rows_of((2, 20000), torch.bfloat16, 4).cuda()
    y, h, _ = ops.rms_norm(long, residual=res)
    y2, h2, _ = ops.rms_norm(long, residual=res, h_out=res)
    assert torch.equal(h, res) and torch.equal(y, y2)
    e = ops.rms_norm(base[:0, 0])
    assert e[0].shape == (0, 700) and e[2].shape == (0,)
    # rows of zeros: zeros with eps, and what the formula says without
    z = torch.zeros((3, 40), device="cuda")
    assert not ops.rms_norm(z, eps=1e-6)[0].any()
    assert torch.isnan(ops.rms_norm(z, eps=0.0)[0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 8), (9, 30), (5, 128), (4, 200), (7, 513), (5, 1000), (3, 2056),
                                       (2, 8192), (2, 16384), (2, 17000)])
@pytest.mark.parametrize("group", [0, 8, 32, 128, 512])
def test_rms_norm_8bit(cuda_device, dtype, rows, cols, group):
    x, w = rows_of((rows, cols), dtype, 1), rows_of((cols,), dtype, 2) + 1
    r = rows_of((rows, cols), dtype, 3, 4.0)
    y, h, rstd, off = want_norm(x, w, 1e-6, r, None)
    q, scales, gh = ops.rms_norm_8bit(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), group=group)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (rows, cols)
    g = group or cols
    groups = -(-cols // g)
    assert scales.shape == (rows, groups)
    rel = rstd_bound(h, off, rstd)[:, None]
    ybound = y.abs() * (rel + 3 * U) + off * rstd[:, None] * w.double().abs()
    pad = torch.nn.functional.pad
    top = pad(y.abs(), (0, -cols % g)).view(rows, groups, g).amax(2)
    slack = pad(ybound, (0, -cols % g)).view(rows, groups, g).amax(2)
    within(scales, top / 448, (slack + top * U) / 448)
    # a value's share of its scale, rounded to e4m3: half a step relative, or half of the smallest step 2^-9
    each = scales.double().cpu().repeat_interleave(g, 1)[:, :cols]
    within(q.float().double().cpu() * each, y, ybound + (2 ** -4 + 2 * U) * (y.abs() + ybound) + 2.0 ** -10 * each)
    # the group's largest value is the type's largest
    unit = pad(q.float().abs().cpu(), (0, -cols % g)).view(rows, groups, g).amax(2)
    assert bool((unit == 448).all())
    within(gh, h, off + half_step(dtype) * (h.abs() + off))


def test_rms_norm_forms_agree(cuda_device):
    """One row without a row dimension, a copy of h without residual, and the 8-bit form with dropout."""
    x, w = rows_of((300,), torch.bfloat16, 1).cuda(), rows_of((300,), torch.float32, 2).cuda()
    y, h, rstd = ops.rms_norm(x, w)
    y2, h2, rstd2 = ops.rms_norm(x.view(1, 300), w, h_out=torch.empty((1, 300), dtype=torch.bfloat16, device="cuda"))
    assert rstd.shape == () and torch.equal(y, y2[0]) and torch.equal(h2[0], x) and torch.equal(rstd, rstd2[0])
    gx, gr, gw = ops.rms_norm_grad(y, h, w, rstd)
    gx2, _, gw2 = ops.rms_norm_grad(y2, h2, w, rstd2, residual_grad=False)
    assert torch.equal(gx, gx2[0]) and torch.equal(gw, gw2)
    q, scales, h = ops.rms_norm_8bit(x, w, group=64)
    assert q.shape == (300,) and scales.shape == (5,) and h is x
    x, res, drop = rows_of((40, 300), torch.bfloat16, 3).cuda(), rows_of((40, 300), torch.float32, 4).cuda(), (0.3, 4, 5)
    y, h, _ = ops.rms_norm(x, w, residual=res, dropout=drop)
    q, scales, h8 = ops.rms_norm_8bit(x, w, residual=res, dropout=drop)
    assert torch.equal(h, h8)
    # y is rounded to bfloat16, q to e4m3 in units of the scale; both from the same float32 value
    bound = y.double().abs() * (2 ** -8 + 2 ** -4 + 2 ** -11) + 2.0 ** -10 * scales.double()
    within(q.float().double() * scales.double(), y, bound)
    y, h, _ = ops.rms_norm(x, w, dropout=drop)
    assert torch.equal(h, ops.dropout(x, *drop))


@pytest.mark.parametrize("rows,cols", [(64, 512), (7, 1001), (33, 4096), (2, 17_000)])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("size", [1.0, 1e-12, 1e-25, 1e28, 1e33])
def test_rms_norm_8bit_rounds_the_quotient(cuda_device, rows, cols, group, size):
    """The float32 form gives the same y, so scale and quotient can be looked at alone.  scale: a product and a
    correction, one step of 2^-23 at most.  q: half a step of e4m3, 2^-4 of the power of two below the value and at
    least 2^-10, and two steps of float32 beside a tie (the quotient's rounding and the correction's)."""
    x, w = rows_of((rows, cols), torch.float32, 11).cuda(), (rows_of((cols,), torch.float32, 12) * size).cuda()
    y = ops.rms_norm(x, w)[0].double().cpu()
    q, scales, _ = ops.rms_norm_8bit(x, w, group=group)
    g = group or cols
    top = torch.nn.functional.pad(y.abs(), (0, -cols % g)).view(rows, -1, g).amax(2)
    within(scales, top / 448, top / 448 * 2.0 ** -23)
    u = y / scales.double().cpu().repeat_interleave(g, 1)[:, :cols]
    half = torch.exp2(u.abs().clamp_min(2.0 ** -6).log2().floor()) * 2.0 ** -4
    within(q.float(), u, half + u.abs() * 2.0 ** -23)


def test_rms_norm_8bit_of_zeros_and_infinities(cuda_device):
    x = rows_of((4, 256), torch.float32, 1)
    x[1] = 0
    x[2, 5] = float("nan")
    q, scales, _ = ops.rms_norm_8bit(x.cuda(), group=128)
    assert not scales[1].any() and not q[1].float().any()
    assert torch.isnan(scales[2]).all() and torch.isfinite(scales[[0, 3]]).all()
    w = torch.ones(256)
    w[200] = float("inf")
    q, scales, _ = ops.rms_norm_8bit(x[:1].cuda(), w.cuda(), group=128)
    assert torch.isfinite(scales[0, 0]) and torch.isinf(scales[0, 1])
    # the smallest magnitudes: scales that are themselves subnormal stay usable
    small = torch.full((1, 64), 1e-3)
    q, scales, _ = ops.rms_norm_8bit(small.cuda(), torch.full((64,), 1e-38).cuda())
    assert bool((q.float() == 448).all())


@pytest.mark.parametrize("dtype,stream,wtype", [
    (torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
    (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float32, torch.float16),
    (torch.float32, torch.float32, None)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (300, 64), (33, 100), (9, 250), (5, 512), (70, 1000), (3, 2048),
                                       (1500, 2049), (4, 8192), (3, 16384), (70, 16400)])
@pytest.mark.parametrize("mode", ["plain", "residual", "dropout"])
def test_rms_norm_grad_against_64_bits(cuda_device, dtype, stream, wtype, rows, cols, mode):
    g, h = rows_of((rows, cols), dtype, 1), rows_of((rows, cols), stream, 2, 3.0)
    w = None if wtype is None else rows_of((cols,), wtype, 3) + 1
    gh = rows_of((rows, cols), stream, 4) if mode != "plain" else None
    drop = (0.2, 77, 5) if mode == "dropout" else None
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    r = rstd.double()[:, None]
    n, a = h.double() * r, g.double() * (1 if w is None else w.double())
    dh = r * (a - n * (a * n).mean(1, keepdim=True)) + (0 if gh is None else gh.double())
    # the mean's terms: cols additions and 4 products; then 5 operations on what is summed here
    size = r * (a.abs() + n.abs() * (a * n).abs().mean(1, keepdim=True)) + (0 if gh is None else gh.double().abs())
    off = U * (8 * size + r * n.abs() * (cols + 4) * (a * n).abs().mean(1, keepdim=True))
    gx, gr, gw = ops.rms_norm_grad(g.cuda(), h.cuda(), None if w is None else w.cuda(), rstd.cuda(),
                                   grad_h=None if gh is None else gh.cuda(), dropout=drop)
    f = factors(rows, cols, drop)
    want = dh * f
    within(gx, want, (off + 2 * U * dh.abs()) * f + half_step(dtype) * (want.abs() + off * f) + tiny(dtype))
    assert gx.dtype == dtype and gr.dtype == stream
    within(gr, dh, off + half_step(stream) * (dh.abs() + off) + tiny(stream))
    if w is None:
        assert gw is None
        return
    assert gw.dtype == wtype
    want, size = (g.double() * n).sum(0), (g.double() * n).abs().sum(0)
    off = (rows + 4) * U * size
    within(gw, want, off + half_step(wtype) * (want.abs() + off) + tiny(wtype))
    again = ops.rms_norm_grad(g.cuda(), h.cuda(), w.cuda(), rstd.cuda(), grad_h=None if gh is None else gh.cuda(),
                              dropout=drop)
    assert torch.equal(gw, again[2]) and torch.equal(gx, again[0])


def test_rms_norm_grad_options_views_and_no_rows(cuda_device):
    base = rows_of((8, 3, 300), torch.bfloat16, 1).cuda()
    g, h = base[:, 0, 1:258], base[:, 1, 7:264]
    w = rows_of((257,), torch.bfloat16, 2).cuda()
    rstd = torch.rand(8, device="cuda") + 0.5
    gx, gr, gw = ops.rms_norm_grad(g, h, w, rstd)
    assert gr is gx
    gx2, gr2, gw2 = ops.rms_norm_grad(g.contiguous(), h.contiguous(), w, rstd, residual_grad=False, weight_grad=False)
    assert torch.equal(gx, gx2) and gr2 is None and gw2 is None
    empty = ops.rms_norm_grad(g[:0], h[:0], w, rstd[:0])
    assert empty[0].shape == (0, 257) and empty[2].shape == (257,) and not empty[2].any()


def test_rms_norm_grad_against_differences(cuda_device):
    """The whole map y, h of x, residual and weight, with dropout, against central differences in 64 bits."""
    rows, cols, eps, drop = 2, 12, 1e-3, (0.3, 9, 1)
    x, r, w = rows_of((rows, cols), torch.float32, 1), rows_of((rows, cols), torch.float32, 2), rows_of((cols,), torch.float32, 3)
    cy, ch = rows_of((rows, cols), torch.float32, 4), rows_of((rows, cols), torch.float32, 5)

    def value(x, r, w):
        y, h, _, _ = want_norm(x, w, eps, r, drop)
        return float((y * cy.double()).sum() + (h * ch.double()).sum())
    y, h, rstd = ops.rms_norm(x.cuda(), w.cuda(), eps, residual=r.cuda(), dropout=drop)
    gx, gr, gw = ops.rms_norm_grad(cy.cuda(), h, w.cuda(), rstd, grad_h=ch.cuda(), dropout=drop)
    at = [x.double(), r.double(), w.double()]
    step = 1e-5
    for k, got in enumerate((gx, gr, gw)):
        want = torch.empty_like(at[k])
        for i in range(at[k].numel()):
            d = []
            for s in (step, -step):
                moved = [t.clone() for t in at]
                moved[k].view(-1)[i] += s
                d.append(value(*moved))
            want.view(-1)[i] = (d[0] - d[1]) / (2 * step)
        # differences: step^2 times a third derivative of a few hundred at most; kernel: float32 chains of
        # about 20 operations on sums of at most 100
        within(got, want, 500 * step ** 2 + 20 * U * 100)


# ---- streams, graphs, far offsets, refusals ---------------------------------------------------------------
def test_offset_on_the_device_and_captured_replays(cuda_device):
    """A captured step - lookup, norm, both gradients - draws a new mask on every replay from the offset that the
    graph itself counts up, and gives what the eager calls give; two graphs do not disturb each other."""
    n, vocab, dim, scale = 300, 90, 257, 3.0
    w = rows_of((vocab, dim), torch.bfloat16, 1).cuda()
    res = rows_of((n, dim), torch.float32, 2).cuda()
    gamma = rows_of((dim,), torch.bfloat16, 3).cuda()
    gy = rows_of((n, dim), torch.bfloat16, 4).cuda()

    def step(ids, offset):
        x = ops.embed(w, ids, scale=scale, dropout=(0.1, 5, offset))
        y, h, rstd = ops.rms_norm(x, gamma, residual=res, dropout=(0.2, 6, offset))
        gx, gr, gg = ops.rms_norm_grad(gy, h, gamma, rstd, dropout=(0.2, 6, offset))
        gw = ops.embed_grad(gx, ids, vocab, scale=scale, dropout=(0.1, 5, offset))
        q, scales, _ = ops.rms_norm_8bit(ops.dropout(x, 0.3, 7, offset), gamma, group=64)
        return [x, y, h, gx, gr, gg, gw, q.view(torch.uint8), scales]

    graphs = []
    for k in range(2):
        ids = token_ids(n, vocab, 10 + k, 0.1).cuda()
        offset = torch.zeros(1, dtype=torch.int64, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(ids, offset)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ids, offset)
            offset.add_(1)
        graphs.append((graph, ids, offset, outs))
    for turn in range(4):
        for k, (graph, ids, offset, outs) in enumerate(graphs):
            ids.copy_(token_ids(n, vocab, 20 + turn + 7 * k, 0.1))
            graph.replay()
            want = step(ids, turn)
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
            assert int(offset) == turn + 1


def test_calls_on_two_streams_at_once(cuda_device):
    n, vocab, dim = 4000, 500, 256
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    data = [(rows_of((n, dim), torch.bfloat16, k).cuda(), token_ids(n, vocab, k).cuda()) for k in range(2)]
    want = [ops.embed_grad(g, ids, vocab) for g, ids in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(ops.embed_grad(*data[k], vocab))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k]) for k in range(2) for g in got[k])


def test_offsets_past_32_bits(cuda_device):
    """Rows that lie more than 2^31 elements (and 2^32 bytes) into their tensors."""
    dim, vocab = 8192, 300_000                              # 2.46e9 values
    table = torch.zeros((vocab, dim), dtype=torch.bfloat16, device="cuda")
    last = rows_of((3, dim), torch.bfloat16, 1).cuda()
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 3], device="cuda")
    table[vocab - 3:] = last
    got = ops.embed(table, ids)
    assert torch.equal(got[[3, 2, 0]], last) and not got[1].any()
    grad = ops.embed_grad(got, ids, vocab, out=table)
    assert torch.equal(grad[vocab - 3:], last) and not grad[:vocab - 3].any()
    # the same rows as a batch: a mask and a norm at the end of the tensor
    drop = (0.5, 3, 4)
    table[vocab - 3:] = last
    out = ops.dropout(table, *drop)
    f = factors(np.arange(vocab - 3, vocab), dim, drop)
    want = last.double().cpu() * f
    within(out[vocab - 3:], want, want.abs() * (2 * U + half_step(torch.bfloat16)))
    assert not out[:vocab - 3].any()
    y, h, rstd = ops.rms_norm(table, residual=out, h_out=out)
    small = ops.rms_norm(table[vocab - 3:], residual=want.to(torch.bfloat16).cuda())
    assert torch.equal(y[vocab - 3:], small[0]) and torch.equal(rstd[vocab - 3:], small[2])
    gx, gr, _ = ops.rms_norm_grad(y, h, None, rstd, dropout=drop)
    part = ops.rms_norm_grad(y[vocab - 3:], h[vocab - 3:], None, rstd[vocab - 3:])
    assert torch.equal(gr[vocab - 3:], part[1])
    within(gx[vocab - 3:], gr[vocab - 3:].double().cpu() * f, gr[vocab - 3:].double().cpu().abs() * 2 ** -6 + 1e-30)


def test_more_than_2_to_31_pieces(cuda_device):
    """A dropout in place over 2^34 values and more: the flat list of pieces passes 31 bits."""
    rows, cols = (1 << 21) + 3, 8192
    x = torch.ones((rows, cols), dtype=torch.bfloat16, device="cuda")
    assert ops.dropout(x, 0.5, 1, 2, out=x) is x
    for at in (0, rows // 2, rows - 1):
        assert torch.equal(x[at:at + 1].double().cpu(), factors(np.arange(at, at + 1), cols, (0.5, 1, 2)))


def test_refusals_on_device_tensors(cuda_device):
    x = torch.zeros((4, 8), device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    w = torch.ones(8, device="cuda")
    rstd = torch.ones(4, device="cuda")
    bad = [
        (lambda: ops.embed(x.double(), ids), "float, half"),
        (lambda: ops.embed(x, ids.short()), "int32 or int64"),
        (lambda: ops.embed(x, ids.cpu()), "ids must be"),
        (lambda: ops.embed(x, torch.zeros((4, 2), dtype=torch.int64, device="cuda")[:, 0]), "contiguous"),
        (lambda: ops.embed(x.t(), ids), "rows must be contiguous"),
        (lambda: ops.embed(x[0].expand(4, 8), ids), "overlap"),
        (lambda: ops.embed(x[0], ids), "num_rows, dim"),
        (lambda: ops.embed(x, ids, out=x[:3]), "wrong shape"),
        (lambda: ops.embed(x, ids, dropout=(1.5, 0, 0)), "p must lie"),
        (lambda: ops.embed(x, ids, dropout=(0.5, 1 << 64, 0)), "seed"),
        (lambda: ops.embed(x, ids, dropout=(0.5, 0, -1)), "offset"),
        (lambda: ops.embed(x, ids, dropout=(0.5, 0, torch.zeros(1, dtype=torch.int64))), "offset must be"),
        (lambda: ops.embed_grad(x, ids[:3], 4), "one row per id"),
        (lambda: ops.embed_grad(x, ids, 4, accumulate=True), "needs out"),
        (lambda: ops.embed_grad(x, ids, 4, padding_idx=4), "padding_idx"),
        (lambda: ops.embed_grad(x, ids, 4, out=x.half()), "rows' or float"),
        (lambda: ops.embed_grad(x, ids, 5, out=x), "wrong shape"),
        (lambda: ops.dropout(x, 0.5, 1, 2, residual=x.half()), "residual"),
        (lambda: ops.dropout(x[0, 0], 0.5, 1, 2), "dimension"),
        (lambda: ops.dropout(x, float("nan"), 1, 2), "p must lie"),
        (lambda: ops.rms_norm(x, w[:7]), "weight must be"),
        (lambda: ops.rms_norm(x, w.half()), "weight must be"),
        (lambda: ops.rms_norm(x.half(), residual=x.bfloat16()), "residual must"),
        (lambda: ops.rms_norm(x, eps=-1.0), "eps"),
        (lambda: ops.rms_norm(x[:, :0]), "at least one value"),
        (lambda: ops.rms_norm(x, out=x.half()), "wrong shape/dtype"),
        (lambda: ops.rms_norm_8bit(x, group=100), "group"),
        (lambda: ops.rms_norm_grad(x, x.half(), w, rstd), "h must have"),
        (lambda: ops.rms_norm_grad(x, x, w, rstd[:3]), "rstd"),
        (lambda: ops.rms_norm_grad(x, x, w, rstd, grad_h=x.half()), "grad_h"),
    ]
    for call, match in bad:
        with pytest.raises(RuntimeError, match=match):
            call()
