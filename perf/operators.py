"""The operators of a model's input stage, as they are measured: embedding lookup with scaling and its
gradient by sorted tokens, dropout from a counter-based generator, and the root-mean-square norm with the
residual's addition, an output in 8 bits and its gradient.

`run` computes a case in elementary torch operations (`own = False`) or through hades_amd's entry points
(`own = True`); `exact` gives the same results from the definitions in 64 bits, written apart from `run`.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # a server's step for one sequence: one token's row, where the call itself is the cost
        {"name": "embed one token", "op": "embed", "n": 1, "vocab": 32000, "dim": 4096, "dtype": "bfloat16",
         "ids": "int64", "scale": 64.0, "p": 0.0},
        # a fine-tuning batch on a float32 table whose rows are not a whole number of 16-byte pieces
        {"name": "embed odd rows", "op": "embed", "n": 3001, "vocab": 50257, "dim": 1001, "dtype": "float32",
         "ids": "int32", "scale": 1.0, "p": 0.1},
        # a training batch of a wide model: scaled rows with dropout
        {"name": "embed batch", "op": "embed", "n": 32768, "vocab": 131072, "dim": 4096, "dtype": "bfloat16",
         "ids": "int64", "scale": 64.0, "p": 0.1},
        # the gradient of a small model's step: the sort and the launches count
        {"name": "embed_grad small", "op": "embed_grad", "n": 2048, "vocab": 32000, "dim": 1024,
         "dtype": "float32", "ids": "int64", "scale": 1.0, "p": 0.0, "pad": 0.0},
        # a padded batch of odd lengths: a tenth of the positions hold no token
        {"name": "embed_grad padded", "op": "embed_grad", "n": 12289, "vocab": 50257, "dim": 1001,
         "dtype": "float16", "ids": "int64", "scale": 8.0, "p": 0.0, "pad": 0.1},
        # the gradient of the wide model's batch, its dropout mask drawn again from the counters
        {"name": "embed_grad batch", "op": "embed_grad", "n": 32768, "vocab": 131072, "dim": 4096,
         "dtype": "bfloat16", "ids": "int64", "scale": 64.0, "p": 0.1, "pad": 0.0},
        # a small layer's backward pass with odd rows
        {"name": "dropout_grad odd", "op": "dropout_grad", "rows": 777, "cols": 1111, "dtype": "float16",
         "p": 0.3, "residual": False},
        # a layer's output dropped and added to the residual stream
        {"name": "dropout batch", "op": "dropout", "rows": 32768, "cols": 4096, "dtype": "bfloat16",
         "p": 0.1, "residual": True},
        # one decoding step of sixteen sequences
        {"name": "rms_norm tokens", "op": "rms_norm", "rows": 16, "cols": 4096, "dtype": "bfloat16",
         "stream": "bfloat16", "p": 0.0, "residual": True},
        # a prompt's rows on their way into an 8-bit matrix product
        {"name": "rms_norm_8bit prompt", "op": "rms_norm_8bit", "rows": 16384, "cols": 8192,
         "dtype": "bfloat16", "stream": "bfloat16", "p": 0.0, "residual": True, "group": 128},
        # a small model's gradient, float32 rows of odd width
        {"name": "rms_norm_grad odd", "op": "rms_norm_grad", "rows": 1023, "cols": 333, "dtype": "float32",
         "stream": "float32", "p": 0.0, "residual": False},
        # the gradient of a wide model's layer: residual stream's gradient added, dropout drawn again
        {"name": "rms_norm_grad batch", "op": "rms_norm_grad", "rows": 16384, "cols": 4096,
         "dtype": "bfloat16", "stream": "bfloat16", "p": 0.1, "residual": True},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A row width: two in three a multiple of 64, the others any number."""
    w = _spread(rng, low, high)
    return w if rng.random() < 1 / 3 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "dropout", "dropout_grad", "rms_norm", "rms_norm_8bit", "rms_norm_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    p = rng.choice([0.0, 0.1, round(rng.uniform(0.01, 0.6), 3)])
    width = _width(rng, 64, 8192)
    most = (1 << 27) // (width * _BYTES[dtype] // 2)   # values that the largest listed case's rows hold
    if op in ("embed", "embed_grad"):
        return {"op": op, "n": _spread(rng, 1, min(65536, most)), "vocab": _spread(rng, 1000, min(262144, 2 * most)),
                "dim": width, "dtype": dtype, "ids": rng.choice(["int32", "int64"]),
                "scale": rng.choice([1.0, round(math.sqrt(width), 3)]), "p": p,
                **({"pad": rng.choice([0.0, 0.25])} if op == "embed_grad" else {})}
    rows = _spread(rng, 1, min(65536, most // 2))
    if op in ("dropout", "dropout_grad"):
        return {"op": op, "rows": rows, "cols": width, "dtype": dtype, "p": p or 0.1,
                "residual": op == "dropout" and rng.random() < 0.5}
    case = {"op": op, "rows": rows, "cols": width, "dtype": dtype, "stream": rng.choice([dtype, "float32"]),
            "p": p if op != "rms_norm_8bit" else 0.0, "residual": rng.random() < 0.75}
    if not case["residual"]:
        case.update(stream=dtype, p=0.0)
    if op == "rms_norm_8bit":
        case["group"] = rng.choice([0, 128])
    return case


# ---- inputs ---------------------------------------------------------------------------------------
def _tokens(case, gen):
    """Token ids whose ranks follow a power law (one id in about ln(vocab) is among the two most
    frequent), spread over the table; a share `pad` of the positions holds -1."""
    u = torch.rand(case["n"], generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(case["vocab"] + 1)).long() - 1).clamp_(0, case["vocab"] - 1)
    step = int(case["vocab"] * 0.618) | 1
    while math.gcd(step, case["vocab"]) != 1:
        step += 2
    ids = rank * step % case["vocab"]
    if case.get("pad"):
        ids[torch.rand(case["n"], generator=gen, device="cuda") < case["pad"]] = -1
    return ids.to(getattr(torch, case["ids"]))


def _rows(rows, cols, dtype, gen, scale=1.0, outliers=False):
    x = torch.empty((rows, cols), dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen)
    if outliers:   # a few columns of a residual stream are an order of magnitude larger than the rest
        x[:, ::97] *= 12.0
    return x.to(_DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], case["dtype"]
    s = {"case": case, "seed": seed * 2654435761 % (1 << 63), "offset": seed % 1000 + (1 << 33)}
    if op == "embed":
        s["weight"] = _rows(case["vocab"], case["dim"], dtype, gen, 0.02)
        s["ids"] = _tokens(case, gen)
    elif op == "embed_grad":
        s["ids"] = _tokens(case, gen)
        s["grad"] = _rows(case["n"], case["dim"], dtype, gen, 1e-3 if dtype != "float16" else 0.1)
    elif op in ("dropout", "dropout_grad"):
        s["x"] = _rows(case["rows"], case["cols"], dtype, gen)
        s["residual"] = _rows(case["rows"], case["cols"], dtype, gen, outliers=True) if case["residual"] else None
    else:
        rows, cols, stream = case["rows"], case["cols"], case["stream"]
        s["weight"] = _rows(1, cols, dtype, gen, 0.1)[0] + 1
        if op == "rms_norm_grad":
            s["grad"] = _rows(rows, cols, dtype, gen, 0.1)
            s["h"] = _rows(rows, cols, stream, gen, outliers=True)
            s["grad_h"] = _rows(rows, cols, stream, gen, 0.1) if case["residual"] else None
            s["rstd"] = (s["h"].double().square().mean(1) + EPS).rsqrt().float()
        else:
            s["x"] = _rows(rows, cols, dtype, gen)
            s["residual"] = _rows(rows, cols, stream, gen, outliers=True) if case["residual"] else None
    return s


# ---- the plain forms ------------------------------------------------------------------------------
_M32 = 0xFFFFFFFF


def _threshold(p):
    """Dropout's probability as a whole number of 65536ths."""
    return int(math.floor(p * 65536 + 0.5))


def _keep(rows, cols, p, seed, offset):
    """Where a value is kept: 16 bits for each, from Philox4x32 with 7 rounds (Salmon et al., 2011).  The
    counter is (column / 8, row, offset), the key the seed; products of 32 by 32 bits wrap in int64 as
    unsigned ones do in 64 bits."""
    c0 = torch.arange((cols + 7) // 8, device="cuda").expand(rows, -1)
    c1 = torch.arange(rows, device="cuda").unsqueeze(1).expand(-1, c0.size(1))
    c2 = torch.full_like(c0, offset & _M32)
    c3 = torch.full_like(c0, (offset >> 32) & _M32)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & _M32) ^ c1 ^ k0, b & _M32, (a >> 32 & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    words = torch.stack((c0, c1, c2, c3), -1)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, -1)[:, :cols]
    return halves >= _threshold(p)


def _dropped(x, p, seed, offset):
    """Dropout of float32 rows."""
    if _threshold(p) == 0:
        return x
    s = 65536.0 / (65536 - _threshold(p))
    return torch.where(_keep(x.size(0), x.size(1), p, seed, offset), x * s, torch.zeros_like(x))


def _plain(s):
    case = s["case"]
    op, p, seed, offset = case["op"], case["p"], s["seed"], s["offset"]
    out_type = _DTYPES[case["dtype"]]
    if op == "embed":
        rows = s["weight"][s["ids"].long()].float() * case["scale"]
        return _dropped(rows, p, seed, offset).to(out_type)
    if op == "embed_grad":
        ids = s["ids"].long()
        g = _dropped(s["grad"].float() * case["scale"], p, seed, offset)
        live = ids >= 0
        g = torch.where(live.unsqueeze(1), g, torch.zeros_like(g))
        total = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float32, device="cuda")
        return total.index_add_(0, ids.clamp(min=0), g).to(out_type)
    if op in ("dropout", "dropout_grad"):
        y = _dropped(s["x"].float(), p, seed, offset)
        return (y if s["residual"] is None else y + s["residual"].float()).to(out_type)
    w = s["weight"].float()
    if op == "rms_norm_grad":
        n = s["h"].float() * s["rstd"].unsqueeze(1)
        g = s["grad"].float()
        a = g * w
        dh = s["rstd"].unsqueeze(1) * (a - n * (a * n).mean(1, keepdim=True))
        if s["grad_h"] is not None:
            dh = dh + s["grad_h"].float()
        out = {"grad_x": _dropped(dh, p, seed, offset).to(out_type), "grad_weight": (g * n).sum(0).to(out_type)}
        if s["grad_h"] is not None:
            out["grad_residual"] = dh.to(_DTYPES[case["stream"]])
        return out
    h = _dropped(s["x"].float(), p, seed, offset)
    if s["residual"] is not None:
        h = h + s["residual"].float()
    rstd = torch.rsqrt(h.square().mean(1) + EPS)
    y = h * rstd.unsqueeze(1) * w
    out = {"h": h.to(_DTYPES[case["stream"]])} if s["residual"] is not None else {}
    if op == "rms_norm":
        return {"y": y.to(out_type), "rstd": rstd, **out}
    cols = y.size(1)
    group = case["group"] or cols
    parts = torch.nn.functional.pad(y, (0, -cols % group)).reshape(y.size(0), -1, group)
    scale = parts.abs().amax(2) / E4M3_MAX
    q = torch.where(scale.unsqueeze(2) > 0, parts / scale.unsqueeze(2), torch.zeros_like(parts))
    q = q.clamp(-E4M3_MAX, E4M3_MAX).reshape(y.size(0), -1)[:, :cols].contiguous()
    return {"q": q.to(torch.float8_e4m3fn), "scale": scale, **out}


# ---- the framework's operators --------------------------------------------------------------------
def _own(s):
    from hades_amd import ops
    case = s["case"]
    op, p = case["op"], case["p"]
    drop = (p, s["seed"], s["offset"]) if p else None
    if op == "embed":
        return ops.embed(s["weight"], s["ids"], scale=case["scale"], dropout=drop)
    if op == "embed_grad":
        return ops.embed_grad(s["grad"], s["ids"], case["vocab"], scale=case["scale"], dropout=drop)
    if op == "dropout":
        return ops.dropout(s["x"], p, s["seed"], s["offset"], residual=s["residual"])
    if op == "dropout_grad":
        return ops.dropout_grad(s["x"], p, s["seed"], s["offset"])
    if op == "rms_norm_grad":
        gx, gr, gw = ops.rms_norm_grad(s["grad"], s["h"], s["weight"], s["rstd"], grad_h=s["grad_h"], dropout=drop)
        out = {"grad_x": gx, "grad_weight": gw}
        if s["grad_h"] is not None:
            out["grad_residual"] = gr
        return out
    if op == "rms_norm":
        y, h, rstd = ops.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], dropout=drop)
        out = {"y": y, "rstd": rstd}
    else:
        q, scale, h = ops.rms_norm_8bit(s["x"], s["weight"], EPS, residual=s["residual"], group=case["group"])
        out = {"q": q, "scale": scale}
    if s["residual"] is not None:
        out["h"] = h
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    op, b = case["op"], _BYTES[case["dtype"]]
    if op in ("embed", "embed_grad"):
        n, row = case["n"], case["dim"] * b
        ids = n * (8 if case["ids"] == "int64" else 4)
        if op == "embed":
            return {"bytes": ids + n * row + min(n, case["vocab"]) * row, "flops": n * case["dim"]}
        return {"bytes": ids + n * row + case["vocab"] * row, "flops": 2 * n * case["dim"]}
    values = case["rows"] * case["cols"]
    if op in ("dropout", "dropout_grad"):
        return {"bytes": values * b * (3 if case["residual"] else 2), "flops": 2 * values}
    stream = _BYTES[case["stream"]] if case["residual"] else 0
    if op == "rms_norm":
        return {"bytes": values * (2 * b + 2 * stream), "flops": 5 * values}
    if op == "rms_norm_8bit":
        scales = 4 * case["rows"] * (-(-case["cols"] // case["group"]) if case["group"] else 1)
        return {"bytes": values * (b + 1 + 2 * stream) + scales, "flops": 7 * values}
    own_grad = stream if case["p"] or case["stream"] != case["dtype"] else 0   # else grad_x is the residual's gradient too
    return {"bytes": values * (2 * b + _BYTES[case["stream"]] + stream + own_grad), "flops": 9 * values}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _factors(rows, cols, p, seed, offset):
    """What dropout multiplies each value with, in 64 bits."""
    t = int(np.floor(np.float64(p) * 65536 + 0.5))
    if t == 0:
        return 1.0
    low = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    groups = -(-cols // 8)
    x = [np.tile(np.arange(groups, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), groups),
         np.full(rows * groups, offset & 0xFFFFFFFF, dtype=np.uint64), np.full(rows * groups, offset >> 32, dtype=np.uint64)]
    for i in range(7):
        key = [np.uint64(((seed & 0xFFFFFFFF) + i * 0x9E3779B9) & 0xFFFFFFFF),
               np.uint64(((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)]
        first, second = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(second >> shift) ^ x[1] ^ key[0], second & low, (first >> shift) ^ x[3] ^ key[1], first & low]
    bits = np.empty((rows, groups, 8), dtype=np.uint16)
    for w in range(4):
        bits[:, :, 2 * w] = (x[w] & np.uint64(0xFFFF)).reshape(rows, groups)
        bits[:, :, 2 * w + 1] = (x[w] >> np.uint64(16)).reshape(rows, groups)
    kept = bits.reshape(rows, groups * 8)[:, :cols] >= t
    return torch.from_numpy(np.ascontiguousarray(kept)).cuda().double().mul_(65536 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("embed", "embed_grad"):
        factor = _factors(case["n"], case["dim"], case["p"], s["seed"], s["offset"])
        if op == "embed":
            return torch.index_select(s["weight"], 0, s["ids"].long()).double() * case["scale"] * factor
        order = torch.argsort(s["ids"], stable=True)
        ids = s["ids"].long()[order]
        order = order[ids >= 0]
        total = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device="cuda")
        return total.index_add_(0, ids[ids >= 0], (s["grad"].double() * factor)[order]).mul_(case["scale"])
    factor = _factors(case["rows"], case["cols"], case["p"], s["seed"], s["offset"])
    if op in ("dropout", "dropout_grad"):
        return s["x"].double() * factor + (0.0 if s["residual"] is None else s["residual"].double())
    w = s["weight"].double()
    if op == "rms_norm_grad":
        h, g, r = s["h"].double(), s["grad"].double(), s["rstd"].double()[:, None]
        along = torch.matmul(g * h, w)[:, None] / case["cols"]   # the gradient's part along h
        dh = r * w * g - r.pow(3) * along * h
        if s["grad_h"] is not None:
            dh += s["grad_h"].double()
        out = {"grad_x": dh * factor, "grad_weight": torch.matmul(r[:, 0], g * h)}
        if s["grad_h"] is not None:
            out["grad_residual"] = dh
        return out
    h = s["x"].double() * factor + (0.0 if s["residual"] is None else s["residual"].double())
    rstd = 1.0 / torch.sqrt((h * h).sum(1) / case["cols"] + EPS)
    y = h * (rstd[:, None] * w)
    out = {} if s["residual"] is None else {"h": h}
    if op == "rms_norm":
        return {"y": y, "rstd": rstd, **out}
    group = case["group"] or case["cols"]
    scales = torch.stack([part.abs().max(1).values for part in y.split(group, 1)], 1) / E4M3_MAX
    unit = y / torch.repeat_interleave(scales, group, 1)[:, : case["cols"]].clamp(min=1e-300)
    return {"q": unit.to(torch.float8_e4m3fn).double(), "scale": scales, **out}
