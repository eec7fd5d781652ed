"""Workloads of the joint network's layers in training and decoding: Dense with its epilogue, dropout, one beam step.

  dense        y = residual + dropout(act(x W + b)), forward alone (a decoder's call) or with its backward pass
  dropout      Philox4x32-10 mask that is recomputed in the backward pass, never stored
  beam         selection over beams x vocabulary, then the hypotheses' states in their new order

Every pass is computed here in plain torch (`own` false) or by the package's operators (`own` true).
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the last joint layer for one utterance's beam: 250 hidden units to the 62 symbols of TIMIT; pure latency
        {"name": "dense decode 8x250x62 fp32", "op": "dense", "train": False, "rows": 8, "k": 250, "n": 62, "dtype": "fp32",
         "act": "linear", "bias": True, "residual": False, "rate": 0.0},
        # a batch of beams through a wide output layer: the weights are read once for 64 rows
        {"name": "dense decode 64x2048x8192 bf16", "op": "dense", "train": False, "rows": 64, "k": 2048, "n": 8192, "dtype": "bf16",
         "act": "linear", "bias": True, "residual": False, "rate": 0.0},
        # a hidden layer with a skip connection over the frames of a batch, inference in the library's default type
        {"name": "dense 12800x1024x1024 fp32", "op": "dense", "train": False, "rows": 12800, "k": 1024, "n": 1024, "dtype": "fp32",
         "act": "tanh", "bias": True, "residual": True, "rate": 0.0},
        # joint layer of a TIMIT batch in training: B=8, T=150, U+1=41 positions, 250 hidden units, tanh and dropout
        {"name": "train 49200x250x250 fp32", "op": "dense", "train": True, "rows": 49200, "k": 250, "n": 250, "dtype": "fp32",
         "act": "tanh", "bias": True, "residual": False, "rate": 0.2},
        # odd sizes everywhere, a skip connection and dropout, half precision
        {"name": "train 6151x515x1030 fp16", "op": "dense", "train": True, "rows": 6151, "k": 515, "n": 1030, "dtype": "fp16",
         "act": "silu", "bias": True, "residual": True, "rate": 0.3},
        # the widening layer of a feed-forward block over a large training batch: the largest case
        {"name": "train 32768x1024x4096 bf16", "op": "dense", "train": True, "rows": 32768, "k": 1024, "n": 4096, "dtype": "bf16",
         "act": "gelu", "bias": True, "residual": False, "rate": 0.1},
        # noise on the frames of a TIMIT batch
        {"name": "dropout 1200x250 fp32", "op": "dropout", "rows": 1200, "n": 250, "dtype": "fp32", "rate": 0.5},
        # noise on the hidden layer over a whole lattice, in half the bytes
        {"name": "dropout 262144x1024 bf16", "op": "dropout", "rows": 262144, "n": 1024, "dtype": "bf16", "rate": 0.1},
        # one utterance, four hypotheses, TIMIT's symbols, a 3-layer 250-unit prediction network: latency
        {"name": "beam 1x4x62 fp32", "op": "beam", "batch": 1, "beams": 4, "width": 4, "vocab": 62, "dtype": "fp32", "enc": True,
         "mask": False, "finished": True, "layers": 3, "hidden": 250},
        # a batch of utterances over a word-piece vocabulary
        {"name": "beam 64x8x1024 fp32", "op": "beam", "batch": 64, "beams": 8, "width": 8, "vocab": 1024, "dtype": "fp32", "enc": True,
         "mask": False, "finished": True, "layers": 2, "hidden": 1024},
        # a large vocabulary of odd size with some symbols forbidden per utterance
        {"name": "beam 32x16x32003 bf16", "op": "beam", "batch": 32, "beams": 16, "width": 16, "vocab": 32003, "dtype": "bf16", "enc": False,
         "mask": True, "finished": False, "layers": 2, "hidden": 640},
        # few rows of a very large vocabulary, wide beam, and states that outweigh the logits
        {"name": "beam 4x32x65536 fp16", "op": "beam", "batch": 4, "beams": 32, "width": 32, "vocab": 65536, "dtype": "fp16", "enc": False,
         "mask": False, "finished": True, "layers": 8, "hidden": 4096},
    ]


_MOST_FLOPS = 6.0 * 32768 * 1024 * 4096
_MOST_VALUES = 262144 * 1024
_MOST_LOGITS = 32 * 16 * 32003
_MOST_STATE = 2 * 8 * 4 * 32 * 4096


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v -= v % rng.choice((8, 32, 64))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("dense", "dense", "dense", "dropout", "beam", "beam"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    while True:
        if op == "dense":
            train = rng.random() < 0.5
            c = {"op": op, "train": train, "rows": _log_int(rng, 1, 65536), "k": _log_int(rng, 8, 8192), "n": _log_int(rng, 8, 8192),
                 "dtype": dtype, "act": rng.choice(("linear", "tanh", "relu", "gelu", "silu")), "bias": rng.random() < 0.8,
                 "residual": rng.random() < 0.4, "rate": rng.choice((0.0, 0.1, 0.25)) if train else 0.0}
            # fp32 products cost the plain form and the kernel several times a 16-bit one
            if work(c)["flops"] * (4 if dtype == "fp32" else 1) <= _MOST_FLOPS:
                return c
        elif op == "dropout":
            c = {"op": op, "rows": _log_int(rng, 1, 262144), "n": _log_int(rng, 16, 8192), "dtype": dtype, "rate": rng.choice((0.05, 0.1, 0.3, 0.5))}
            if c["rows"] * c["n"] * SIZE[dtype] <= 2 * _MOST_VALUES:
                return c
        else:
            beams = _log_int(rng, 1, 32)
            c = {"op": op, "batch": _log_int(rng, 1, 128), "beams": beams, "width": beams if rng.random() < 0.7 else _log_int(rng, 1, 32),
                 "vocab": _log_int(rng, 40, 65536), "dtype": dtype, "enc": rng.random() < 0.5, "mask": rng.random() < 0.4,
                 "finished": rng.random() < 0.5, "layers": rng.randint(1, 4), "hidden": _log_int(rng, 64, 2048)}
            if c["batch"] * beams * c["vocab"] <= _MOST_LOGITS and 2 * c["layers"] * c["batch"] * max(beams, c["width"]) * c["hidden"] <= _MOST_STATE:
                return c


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "dense":
        m, k, n = case["rows"], case["k"], case["n"]
        once = m * k + k * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)  # x, kernel, bias, residual
        if not case["train"]:
            return {"bytes": s * (once + m * n), "flops": 2.0 * m * k * n}
        grads = m * k + k * n + (n if case["bias"] else 0)
        return {"bytes": s * (once + 2 * m * n + grads), "flops": 6.0 * m * k * n}  # + y, dy
    if case["op"] == "dropout":
        return {"bytes": 4 * s * case["rows"] * case["n"], "flops": 0}  # x, dy, y, dx
    b, k, w, v = case["batch"], case["beams"], case["width"], case["vocab"]
    states = 2 * s * case["layers"] * b * w * case["hidden"] * 2  # h and c, read and written
    return {"bytes": s * b * k * v + (s * b * v if case["enc"] else 0) + (b * v if case["mask"] else 0) + 4 * b * k + 12 * b * w + states,
            "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    t = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(t)

    if case["op"] == "dense":
        m, k, n = case["rows"], case["k"], case["n"]
        st = {"case": case, "x": normal(m, k), "kernel": normal(k, n, scale=k ** -0.5), "bias": normal(n, scale=0.1) if case["bias"] else None,
              "residual": normal(m, n) if case["residual"] else None, "seed": int(seed) * 3 + 1, "offset": int(seed) + 5}
        if case["train"]:
            st["dy"] = normal(m, n, scale=m ** -0.5)
            for p in ("x", "kernel", "bias"):
                if st[p] is not None:
                    st[p].requires_grad_(True)
        return st
    if case["op"] == "dropout":
        m, n = case["rows"], case["n"]
        return {"case": case, "x": normal(m, n).requires_grad_(True), "dy": normal(m, n, scale=m ** -0.5), "seed": int(seed) * 3 + 1, "offset": int(seed) + 5}
    b, k, v = case["batch"], case["beams"], case["vocab"]
    st = {"case": case, "logits": normal(b, k, v, scale=3.0), "enc": normal(b, v, scale=2.0) if case["enc"] else None,
          "scores": torch.rand((b, k), generator=g, device=DEV).mul_(-6.0).sub_(20.0).sort(dim=1, descending=True).values, "end": v // 2,
          "allowed": torch.rand((b, v), generator=g, device=DEV) < 0.9 if case["mask"] else None,
          "finished": torch.rand((b, k), generator=g, device=DEV) < 0.2 if case["finished"] else None,
          "states": [normal(case["layers"], b, k, case["hidden"]) for _ in range(2)]}
    if k > 1 and b > 1:
        st["scores"][0, 1:] = -math.inf  # an utterance at its first step: one hypothesis, the other beams empty
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    return _dense(st) if op == "dense" else _dropout(st) if op == "dropout" else _beam(st)


def _dense(st):
    c = st["case"]
    if own:
        import rnnt_amd
        y = rnnt_amd.dense(st["x"], st["kernel"], st["bias"], activation=c["act"], residual=st["residual"], dropout=c["rate"],
                           seed=st["seed"], offset=st["offset"])
        if not c["train"]:
            return {"y": y}
        leaves = ["x", "kernel"] + (["bias"] if c["bias"] else [])
        grads = torch.autograd.grad(y, [st[p] for p in leaves], st["dy"])
        return {"y": y, **{"d" + p: d for p, d in zip(leaves, grads)}}
    with torch.no_grad():
        t = st["x"].dtype
        x, w = st["x"].float(), st["kernel"].float()
        z = x @ w
        if st["bias"] is not None:
            z = z + st["bias"].float()
        y = _act(z, c["act"])
        scale = _mask_scale(c["rows"], c["n"], c["rate"], st["seed"], st["offset"]) if c["rate"] else None
        if scale is not None:
            y = y * scale
        if st["residual"] is not None:
            y = y + st["residual"].float()
        if not c["train"]:
            return {"y": y.to(t)}
        dz = st["dy"].float()
        if scale is not None:
            dz = dz * scale
        if c["act"] != "linear":
            dz = dz * _act_grad(z, c["act"])
        out = {"y": y.to(t), "dx": (dz @ w.t()).to(t), "dkernel": (x.t() @ dz).to(t)}
        if c["bias"]:
            out["dbias"] = dz.sum(0).to(t)
        return out


def _act(z, act):
    if act == "tanh":
        return torch.tanh(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "tanh":
        a = torch.tanh(z)
        return 1 - a * a
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    p = 1 / (1 + torch.exp(-z))  # silu
    return p * (1 + z * (1 - p))


def _mask_scale(rows, n, rate, seed, offset):
    """[rows, n] float32: 0 where an element is dropped, 1/keep elsewhere. Eight columns share one Philox4x32-10 counter
    (column // 8, row, offset low, offset high) under the key (seed low, seed high); 16 bits decide each."""
    low = 0xFFFFFFFF
    groups = (n + 7) // 8
    c0 = torch.arange(groups, device=DEV).unsqueeze(0).expand(rows, groups)
    c1 = torch.arange(rows, device=DEV).unsqueeze(1).expand(rows, groups)
    c2, c3 = torch.full_like(c0, offset & low), torch.full_like(c0, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wraps modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), dim=-1)
    u = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, groups * 8)[:, :n]
    drop = int(round(rate * 65536))
    return (u >= drop).float() * (65536.0 / (65536 - drop))


def _dropout(st):
    c = st["case"]
    if own:
        import rnnt_amd
        y = rnnt_amd.dropout(st["x"], c["rate"], seed=st["seed"], offset=st["offset"])
        return {"y": y, "dx": torch.autograd.grad(y, st["x"], st["dy"])[0]}
    with torch.no_grad():
        scale = _mask_scale(c["rows"], c["n"], c["rate"], st["seed"], st["offset"])
        t = st["x"].dtype
        return {"y": (st["x"].float() * scale).to(t), "dx": (st["dy"].float() * scale).to(t)}


def _beam(st):
    c = st["case"]
    if own:
        import rnnt_amd
        scores, parent, token = rnnt_amd.beam_select(st["logits"], st["scores"], c["width"], enc=st["enc"], allowed=st["allowed"],
                                                     finished=st["finished"], end=st["end"])
        h, cc = rnnt_amd.beam_reorder(parent, st["states"], batch_dim=1)
        return {"scores": scores, "parent": parent, "token": token, "h": h, "c": cc}
    b, k, v = st["logits"].shape
    x = st["logits"].float()
    if st["enc"] is not None:
        x = x + st["enc"].float().unsqueeze(1)  # the joint's sum is a 32-bit value
    if st["allowed"] is not None:
        x = torch.where(st["allowed"].unsqueeze(1), x, torch.full_like(x, -math.inf))
    x = x.double()  # candidates of different beams lie next to each other: the order is decided in 64 bits
    m = x.amax(dim=2, keepdim=True)
    total = st["scores"].double().unsqueeze(2) + (x - (m + torch.log(torch.exp(x - m).sum(dim=2, keepdim=True))))
    if st["finished"] is not None:
        carried = torch.full_like(total, -math.inf)
        carried[:, :, st["end"]] = st["scores"].double()
        total = torch.where(st["finished"].unsqueeze(2), carried, total)
    best, flat = torch.sort(total.reshape(b, k * v), dim=1, descending=True, stable=True)
    width = min(c["width"], k * v)
    best, flat = best[:, :width], flat[:, :width]
    there = best > -math.inf
    parent = torch.where(there, flat // v, torch.full_like(flat, -1))
    token = torch.where(there, flat % v, torch.full_like(flat, -1))
    pick = torch.arange(b, device=DEV).unsqueeze(1)
    moved = [torch.where(there.unsqueeze(0).unsqueeze(3), s[:, pick, parent.clamp(min=0)], torch.zeros_like(s[:1, :1, :1])) for s in st["states"]]
    return {"scores": best.float(), "parent": parent.int(), "token": token.int(), "h": moved[0], "c": moved[1]}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def _draws(first, end, n, seed, offset):
    """The 16-bit draws of rows first..end-1 and n columns, with every product of two words made of 16-bit halves."""
    groups = -(-n // 8)
    row = torch.arange(first, end, device=DEV).repeat_interleave(groups)
    zero = torch.zeros_like(row)
    x = [torch.arange(groups, device=DEV).repeat(end - first), row, zero + offset % 2 ** 32, zero + offset // 2 ** 32]

    def halves(a, m):  # high and low word of a * m, both factors below 2^32
        al, ah, ml, mh = a % 65536, a // 65536, m % 65536, m // 65536
        low = al * ml
        middle = al * mh + low // 65536
        other = ah * ml + middle % 65536
        return ah * mh + middle // 65536 + other // 65536, (other % 65536) * 65536 + low % 65536

    for r in range(10):
        (h0, l0), (h1, l1) = halves(x[0], 0xD2511F53), halves(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ ((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x[3] ^ ((seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32), l0]
    return torch.cat([h.unsqueeze(1) for w in x for h in (w % 65536, w // 65536)], dim=1).reshape(end - first, groups * 8)[:, :n]


def _kept(rows, n, rate, seed, offset):
    """0 or 1/keep, a block of rows at a time."""
    drop = round(rate * 2 ** 16)
    out = torch.empty((rows, n), dtype=torch.float64, device=DEV)
    block = max(1, (1 << 25) // n)
    for r in range(0, rows, block):
        e = min(rows, r + block)
        out[r:e] = (_draws(r, e, n, seed, offset) >= drop).double() * (2.0 ** 16 / (2 ** 16 - drop))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "dropout":
            s = _kept(case["rows"], case["n"], case["rate"], st["seed"], st["offset"])
            return {"y": st["x"].double() * s, "dx": st["dy"].double() * s}
        return _exact_dense(case, st) if case["op"] == "dense" else _exact_beam(case, st)


def _exact_dense(c, st):
    x, w = st["x"].double(), st["kernel"].double()
    z = torch.mm(x, w)
    if c["bias"]:
        z += st["bias"].double()
    half = torch.special.erfc(-z / math.sqrt(2.0)) / 2  # the normal distribution's function
    act, slope = {
        "linear": lambda: (z, torch.ones_like(z)),
        "tanh": lambda: (torch.tanh(z), 1 / torch.cosh(z) ** 2),
        "relu": lambda: (z.clamp(min=0), torch.sign(z).clamp(min=0)),
        "gelu": lambda: (z * half, half + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
        "silu": lambda: (z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)),
    }[c["act"]]()
    kept = _kept(c["rows"], c["n"], c["rate"], st["seed"], st["offset"]) if c["rate"] else 1.0
    out = {"y": act * kept + (st["residual"].double() if c["residual"] else 0.0)}
    if c["train"]:
        up = st["dy"].double() * kept * slope
        out["dx"], out["dkernel"] = torch.mm(up, w.t()), torch.mm(x.t(), up)
        if c["bias"]:
            out["dbias"] = up.sum(dim=0)
    return out


def _exact_beam(c, st):
    b, k, v = st["logits"].shape
    dead = torch.tensor(-math.inf, dtype=torch.float64, device=DEV)
    scores, parents, tokens = [], [], []
    for i in range(b):  # an utterance at a time: the best candidate, `width` times over
        x = st["logits"][i].float()
        if c["enc"]:
            x = x + st["enc"][i].float()  # by definition the joint's sum is rounded to 32 bits
        x = x.double()
        if c["mask"]:
            x[:, ~st["allowed"][i]] = dead
        t = torch.log_softmax(x, dim=1) + st["scores"][i].double()[:, None]
        if c["finished"]:
            for j in torch.nonzero(st["finished"][i]).flatten().tolist():
                t[j] = dead
                t[j, st["end"]] = st["scores"][i, j].double()
        t = t.flatten()
        place = torch.arange(k * v, device=DEV)
        row = []
        for _ in range(min(c["width"], k * v)):
            top = t.max()
            at = torch.where(t == top, place, k * v).min()
            row.append((top, at))
            t[at] = dead
        top, at = torch.stack([r[0] for r in row]), torch.stack([r[1] for r in row])
        scores.append(top)
        parents.append(torch.where(top > dead, torch.div(at, v, rounding_mode="floor"), -1))
        tokens.append(torch.where(top > dead, at % v, -1))
    parent = torch.stack(parents)
    moved = []
    for s in st["states"]:
        rows = s.double().permute(1, 2, 0, 3)
        moved.append(torch.stack([torch.stack([rows[i, p] if p >= 0 else torch.zeros_like(rows[i, 0]) for p in parent[i].tolist()]) for i in range(b)]).permute(2, 0, 1, 3))
    return {"scores": torch.stack(scores), "parent": parent.int(), "token": torch.stack(tokens).int(), "h": moved[0].contiguous(), "c": moved[1].contiguous()}
