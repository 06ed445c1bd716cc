"""The input stage's host logic at its edges (no GPU): the seeds that modules draw their masks from, and refusals that
come before the first launch."""
import copy
import ctypes
import gc
import pickle

import pytest
import torch

from hades_amd import _lib, dist_emb


def stage(**kw):
    return dist_emb.InputStage(8, torch.float32, dropout=0.5, device="cpu", **kw)


def seed_of(module):
    return module.draw(offset=0)[1]


def test_modules_without_a_seed_draw_different_masks():
    gc.collect()
    stages = [stage() for _ in range(4)]
    table = dist_emb.TokenEmb(10, 8, torch.float32, dropout=0.5, device="cpu")
    assert [s.seed for s in stages] == [None] * 4                  # none before the first mask
    seeds = [seed_of(s) for s in stages] + [seed_of(table.stage)]
    assert len(set(seeds)) == 5
    assert [seed_of(s) for s in stages] == seeds[:4]               # and they stay
    given = stage(seed=max(seeds) + 1)
    after = stage()
    assert seed_of(given) == max(seeds) + 1 and seed_of(after) not in seeds + [given.seed]
    # layers made by copying one that has not drawn yet; a copy of one that has goes on as its original
    layers = [copy.deepcopy(stages_like) for stages_like in [stage()] * 3]
    assert len({seed_of(s) for s in layers} | set(seeds)) == 8
    assert seed_of(copy.deepcopy(stages[1])) == seeds[1]
    # an unpickled module's seed counts as taken, though __init__ never ran for it
    twin = pickle.loads(pickle.dumps(stages[0]))
    first = stages.pop(0).seed
    gc.collect()
    assert seed_of(twin) == first and seed_of(stage()) != first


def test_a_module_that_is_gone_gives_its_seed_back():
    gc.collect()
    kept = stage()
    seed_of(kept)
    one = stage()
    number = seed_of(one)
    del one
    gc.collect()
    assert seed_of(stage()) == number != kept.seed


def test_seeds_are_kept_with_the_state():
    a = stage()
    a.draw(offset=0)
    state = a.state_dict()
    others = [stage() for _ in range(2)]
    for s in others:
        seed_of(s)
    b, named = stage(), stage(seed=77)
    b.load_state_dict(state)
    named.load_state_dict(state)
    assert b.draw(offset=0) == a.draw(offset=0) and named.seed == 77
    fresh = stage()
    fresh.load_state_dict(stage().state_dict())                    # saved before any mask: nothing to take over
    assert fresh.seed is None
    old = {"_extra_state": {"calls": 5}}                           # a state without a seed
    fresh.load_state_dict(old)
    assert fresh.seed is None and fresh._calls == 5


@pytest.mark.parametrize("training", [True, False])
def test_residuals_that_no_mode_takes(training):
    module = stage(seed=3).train(training)
    x = torch.ones((4, 8))
    for bad in (x[:1], x[0], x.bfloat16(), x.double()):
        with pytest.raises(RuntimeError, match="residual must have"):
            module(x, bad, offset=0)


@pytest.mark.parametrize("n,num_rows,dim,dtype", [(8, (1 << 31) - 1, 1024, _lib.F32),      # 2^39 pieces of zeros
                                                  (100, 100, (1 << 31) - 1, _lib.BF16)])   # slices of the join
def test_embed_grad_too_large_is_refused_before_any_launch(n, num_rows, dim, dtype):
    """The call's size is looked at before the sort runs.  (Nothing behind the pointers is touched: here a launch
    would come back as another error.)"""
    lib, one = _lib.load(), ctypes.c_void_p(256)
    rc = lib.hades_embed_grad(one, dim, one, n, one, dim, num_rows, dim, dtype, dtype, _lib.I64, -1, 0, 1.0, 0.0, 0, 0,
                              ctypes.c_void_p(0), one, 1 << 62, ctypes.c_void_p(0))
    assert rc == 1 and b"too many values" in lib.hades_last_error()


def test_rms_norm_grad_of_too_many_columns_is_refused_before_any_launch():
    lib, one, null = _lib.load(), ctypes.c_void_p(256), ctypes.c_void_p(0)

    def call(rows):
        return lib.hades_rms_norm_grad(one, cols, one, cols, one, one, null, 0, one, null, one, rows, cols, _lib.BF16,
                                       _lib.BF16, _lib.BF16, 0.0, 0, 0, null, one, 1 << 62, null)
    cols = (1 << 28) - 63
    for rows in (0, 3):
        assert call(rows) == 1 and b"too many columns" in lib.hades_last_error()
