"""The input-stage operators' refusals and host logic (no GPU): argument checks of the C ABI come back as
codes and messages before any launch, the Python entry points refuse host tensors and wrong arguments."""
import ctypes

import pytest
import torch

from hades_amd import _lib, dist_emb, ops

NULL = ctypes.c_void_p(0)
ONE = ctypes.c_void_p(256)      # never dereferenced: the checks fail first
DROP = (0.0, 0, 0, NULL)


def refused(name, *args, match, code=1):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code
    assert match in lib.hades_last_error().decode()


def test_embed_refusals():
    ok = [ONE, 64, 100, ONE, 10, ONE, 64, _lib.BF16, _lib.I64, 1.0, *DROP, NULL]

    def bad(at, value, match):
        args = list(ok)
        args[at] = value
        refused("hades_embed", *args, match=match)
    bad(7, _lib.F64, "float, half or bfloat16")
    bad(8, 2, "int32 or int64")
    bad(1, 63, "stride")
    bad(4, -1, "n and num_rows")
    bad(4, 1 << 32, "too large")
    bad(6, 0, "dim")
    bad(0, NULL, "null")
    bad(3, NULL, "null")
    bad(10, 1.5, "[0, 1]")
    bad(10, float("nan"), "[0, 1]")
    assert _lib.load().hades_embed(NULL, 64, 100, NULL, 0, NULL, 64, _lib.F32, _lib.I32, 1.0, *DROP, NULL) == 0


def test_embed_grad_refusals():
    big = 1 << 40
    ok = [ONE, 64, ONE, 10, ONE, 64, 100, 64, _lib.BF16, _lib.F32, _lib.I64, -1, 0, 1.0, *DROP, ONE, big, NULL]

    def bad(at, value, match, code=1):
        args = list(ok)
        args[at] = value
        refused("hades_embed_grad", *args, match=match, code=code)
    bad(8, _lib.F64, "float, half or bfloat16")
    bad(9, _lib.F16, "the rows' or float")
    bad(10, 7, "int32 or int64")
    bad(1, 63, "stride")
    bad(5, 63, "stride")
    bad(3, 1 << 30, "2^30")
    bad(6, 1 << 31, "2^31")
    bad(4, NULL, "null")
    bad(0, NULL, "null")
    bad(14, -0.1, "[0, 1]")
    bad(18, NULL, "workspace too small", 3)
    bad(19, 16, "workspace too small", 3)
    bad(18, ctypes.c_void_p(8), "aligned")
    assert _lib.query("hades_embed_grad_workspace_bytes", 0, 64, 100) > 0
    assert _lib.query("hades_embed_grad_workspace_bytes", -1, 64, 100) == 0
    # a table of no rows, and nothing to add
    lib = _lib.load()
    assert lib.hades_embed_grad(NULL, 64, NULL, 0, NULL, 64, 0, 64, 0, 0, 1, -1, 0, 1.0, *DROP, NULL, 0, NULL) == 0
    assert lib.hades_embed_grad(NULL, 64, NULL, 0, NULL, 64, 5, 64, 0, 0, 1, -1, 1, 1.0, *DROP, NULL, 0, NULL) == 0


def test_dropout_refusals():
    ok = [ONE, 64, NULL, 0, ONE, 10, 64, _lib.F16, 0.5, 1, 2, NULL, NULL]

    def bad(at, value, match):
        args = list(ok)
        args[at] = value
        refused("hades_dropout", *args, match=match)
    bad(7, _lib.F64, "float, half or bfloat16")
    bad(1, 0, "stride")              # overlapping rows, e.g. of an expanded tensor
    bad(2, ONE, "stride")
    bad(5, 1 << 32, "2^32")
    bad(6, -1, ">= 0")
    bad(8, 2.0, "[0, 1]")
    bad(0, NULL, "null")
    assert _lib.load().hades_dropout(NULL, 64, NULL, 0, NULL, 0, 64, 0, 0.5, 1, 2, NULL, NULL) == 0
    assert _lib.load().hades_dropout(NULL, 0, NULL, 0, NULL, 3, 0, 0, 0.5, 1, 2, NULL, NULL) == 0


def test_rms_norm_refusals():
    ok = [ONE, 64, NULL, 0, ONE, ONE, NULL, NULL, ONE, 10, 64, _lib.BF16, _lib.BF16, _lib.F32, 0, 1e-6, *DROP, NULL]

    def bad(at, value, match):
        args = list(ok)
        args[at] = value
        refused("hades_rms_norm", *args, match=match)
    bad(11, _lib.F64, "float, half or bfloat16")
    bad(12, _lib.F16, "residual's type")
    bad(13, _lib.F16, "weight's type")
    bad(10, 0, "cols >= 1")
    bad(1, 63, "stride")
    bad(2, ONE, "stride")
    bad(15, -1.0, "eps")
    bad(15, float("nan"), "eps")
    for group in (4, 24, 1024, -8):
        bad(14, group, "group")
    bad(16, 1.01, "[0, 1]")
    bad(5, NULL, "null")
    assert _lib.load().hades_rms_norm(NULL, 64, NULL, 0, NULL, NULL, NULL, NULL, NULL, 0, 64, 0, 0, 0, 0, 1e-6,
                                      *DROP, NULL) == 0


def test_rms_norm_grad_refusals():
    ok = [ONE, 64, ONE, 64, ONE, ONE, NULL, 0, ONE, NULL, ONE, 1000, 64, _lib.BF16, _lib.BF16, _lib.BF16, *DROP,
          ONE, 1 << 40, NULL]

    def bad(at, value, match, code=1):
        args = list(ok)
        args[at] = value
        refused("hades_rms_norm_grad", *args, match=match, code=code)
    bad(13, _lib.F64, "float, half or bfloat16")
    bad(14, _lib.F16, "residual's type")
    bad(15, _lib.F16, "weight's type")
    bad(12, 0, "cols >= 1")
    bad(1, 63, "stride")
    bad(3, 63, "stride")
    bad(6, ONE, "stride")
    bad(4, NULL, "without a weight")
    bad(8, NULL, "null")
    bad(16, 1.01, "[0, 1]")
    bad(20, NULL, "workspace too small", 3)
    bad(21, 128, "workspace too small", 3)
    bad(20, ctypes.c_void_p(8), "aligned")


def test_host_tensors_are_refused():
    x = torch.zeros((4, 8))
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.embed(x, ids), lambda: ops.embed_grad(x, ids, 4), lambda: ops.dropout(x, 0.5, 1, 0),
                 lambda: ops.dropout_grad(x, 0.5, 1, 0), lambda: ops.rms_norm(x), lambda: ops.rms_norm_8bit(x),
                 lambda: ops.rms_norm_grad(x, x, None, x[:, 0])):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


def test_rms_norm_grad_workspace_query_covers_every_type():
    """The bytes that the query names are enough for rows of any type, whichever needs more of them (checked
    before any launch: the workspace's alignment is looked at after its size, and is wrong here)."""
    lib = _lib.load()
    for cols in (1, 8, 64, 65, 100, 512, 513, 768, 1000, 1024, 2048, 4096, 6144, 6145, 8192, 16384, 16385):
        for rows in (1, 5, 511, 512, 513, 3000, 5000, 1_000_000):
            nbytes = _lib.query("hades_rms_norm_grad_workspace_bytes", rows, cols)
            short = set()
            for dtype in (_lib.F32, _lib.F16, _lib.BF16):
                def call(size):
                    return lib.hades_rms_norm_grad(ONE, cols, ONE, cols, ONE, ONE, NULL, 0, ONE, NULL, ONE, rows, cols,
                                                   dtype, dtype, dtype, *DROP, ctypes.c_void_p(8), size, NULL)
                assert call(nbytes) == 1 and b"aligned" in lib.hades_last_error()
                if nbytes:      # (a few rows need no workspace at all)
                    short.add(call(nbytes - 256))
            assert 3 in short or not nbytes
            assert nbytes or rows < 1000


def test_8bit_rows_go_with_a_norm():
    # on host tensors: the refusal comes before any launch
    emb = dist_emb.TokenEmb(10, 8, torch.float32, device="cpu")
    for call in (lambda: emb.forward_8bit(torch.arange(4)), lambda: emb.stage.forward_8bit(torch.zeros(4, 8))):
        with pytest.raises(RuntimeError, match="goes with norm"):
            call()
