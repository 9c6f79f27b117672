"""Measured cases of the embedding-head operators: ragged products by map, the residual norm with
8-bit rows, and microscaled (4- and 8-bit) rows with their products.

A map's head turns the image embeddings of its detections into map-specific ones
(h = z + W_g z, normalised), and the normalised rows are compared with the map's memory bank.
Rows of all maps come packed, map after map; `off` holds the first row of each map.

`own` false: elementary torch operations in 32 bits.  `own` true: the framework's entry points
(scenemap_b200.products).  Both take what prepare() gives.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EMAX = {4: 2, 8: 8}            # exponent of the largest power of two of e2m1 and e4m3
LARGEST = 65536                # most rows of a case
FLOPS = 6 * 65536 * 1152 * 1152  # the largest listed case


def listed():
    return [
        # one detection against one map's head, the shortest call of a robot's frame loop
        {"name": "head 1 row", "op": "grouped", "type": "bf16", "groups": 1, "empty": 0, "rows": 1, "k": 768, "n": 256},
        # one detection or so in each of 64 maps: every head's weights are read for a row or two
        {"name": "head 64 maps, single rows", "op": "grouped", "type": "bf16", "groups": 64, "empty": 9, "rows": 77, "k": 1152, "n": 512},
        # a frame of 64 maps with up to some tens of detections each
        {"name": "head 64 maps, a frame", "op": "grouped", "type": "f16", "groups": 64, "empty": 3, "rows": 1237, "k": 1152, "n": 1152},
        # a small training step of 13 maps, sizes that no tile divides
        {"name": "head train 13 maps", "op": "grouped_train", "type": "f16", "groups": 13, "empty": 2, "rows": 4099, "k": 1000, "n": 520},
        # a training step over the stored views of 32 maps
        {"name": "head train 32 maps", "op": "grouped_train", "type": "bf16", "groups": 32, "empty": 1, "rows": 65536, "k": 1152, "n": 1152},
        # a new view of one object
        {"name": "norm 1 row", "op": "norm", "type": "bf16", "rows": 1, "k": 1152},
        # every object slot of 64 maps (64 x 1024)
        {"name": "norm all slots", "op": "norm", "type": "bf16", "rows": 65536, "k": 1152},
        # a training step's norm, forward and backward, with an odd number of rows
        {"name": "norm train", "op": "norm_train", "type": "f16", "rows": 20001, "k": 768},
        # the association bank into 4 bits
        {"name": "mx4 bank", "op": "quantise", "type": "bf16", "bits": 4, "rows": 16384, "k": 1152},
        # a frame of 256 detections against one bank in 4 bits, the detections quantised on the way
        {"name": "mx4 scores of a frame", "op": "scores", "type": "bf16", "bits": 4, "groups": 1, "empty": 0, "rows": 256, "k": 1152, "n": 16384},
        # 64 maps, each with a bank of its own in 8 bits and a few detections
        {"name": "mx8 scores 64 maps", "op": "scores", "type": "f32", "bits": 8, "groups": 64, "empty": 5, "rows": 611, "k": 1152, "n": 1024},
        # 32 frames of 256 detections against one bank in one call
        {"name": "mx4 scores of 32 frames", "op": "scores", "type": "bf16", "bits": 4, "groups": 1, "empty": 0, "rows": 8192, "k": 1152, "n": 16384},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.25 else max(8, v // 8 * 8)     # some widths leave rows unaligned


def draw(rng):
    op = rng.choice(["grouped", "grouped_train", "norm", "norm_train", "quantise", "scores"])
    c = {"op": op, "type": rng.choice(["bf16", "f16"] if op.startswith("grouped") else ["bf16", "f16", "f32"])}
    if op in ("norm", "norm_train"):
        c.update(rows=_log(rng, 1, LARGEST), k=_width(rng, 64, 2304))
    elif op == "quantise":
        c.update(bits=rng.choice([4, 8]), rows=_log(rng, 1, LARGEST), k=_width(rng, 64, 2304))
    else:
        if op == "scores":
            c["bits"] = rng.choice([4, 8])
        while True:
            g, rows = _log(rng, 1, 64), _log(rng, 1, LARGEST)
            k, n = _width(rng, 64, 2304), _width(rng, 64, 16384 if op == "scores" else 2304)
            passes = 3 if op == "grouped_train" else 1
            if 2 * passes * rows * k * n <= FLOPS and rows * n <= 8192 * 16384 and g * n * k <= 64 * 1152 * 1152:
                break
        full = max(1, min(rows, g - (g > 3) * rng.randrange(0, g // 3 + 1)))
        c.update(groups=g, empty=g - full, rows=rows, k=k, n=n)
    return c


def _counts(case, seed):
    """Rows of each map: uneven, `empty` of them zero."""
    r = random.Random(seed * 7919 + 13)
    full = case["groups"] - case["empty"]
    w = [0.05 + r.random() ** 2 for _ in range(full)]
    spare = case["rows"] - full
    n = [1 + int(spare * v / sum(w)) for v in w]
    for i in range(case["rows"] - sum(n)):
        n[i % full] += 1
    n += [0] * case["empty"]
    r.shuffle(n)
    return n


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def unit(*shape):                      # image embeddings have unit length
        z = rand(*shape)
        return z / z.square().sum(-1, keepdim=True).sqrt()

    s = {"case": dict(case), "type": t}
    rows, k = case["rows"], case["k"]
    if "groups" in case:
        n = _counts(case, seed)
        s["most"] = max(n)
        off = [0]
        for c in n:
            off.append(off[-1] + c)
        s["off"] = torch.tensor(off, dtype=torch.int32, device="cuda")
        s["x"] = unit(rows, k).to(t)
    if case["op"] in ("grouped", "grouped_train"):
        s["w"] = (rand(case["groups"], case["n"], k) / math.sqrt(k)).to(t)
        if case["op"] == "grouped_train":
            s["dy"] = (0.1 * rand(rows, case["n"])).to(t)
    elif case["op"] in ("norm", "norm_train"):
        s["x"] = (0.02 * rand(rows, k)).to(t)
        s["r"] = unit(rows, k).to(t)
        s["gain"] = 1 + 0.1 * rand(k)
        if case["op"] == "norm_train":
            s["dy"], s["dh"] = (0.1 * rand(rows, k)).to(t), (0.1 * rand(rows, k)).to(t)
    elif case["op"] == "quantise":
        s["x"] = unit(rows, k).to(t)
    else:
        bank = unit(case["groups"] * case["n"], k).to(torch.bfloat16)
        codes, scales, _ = _quantise(bank, case["bits"])
        s["codes"] = codes.reshape(case["groups"], case["n"], -1)
        s["scales"] = scales.reshape(case["groups"], case["n"], -1)
    return s


def _two(e):
    """2^e of whole -127 <= e <= 127 from its bits: the device's power function may be off in the last place."""
    e = e.int()
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


# ---- microscaled rows in plain operations: blocks of 32 along a row share a power of two ----

def _quantise(x, bits):
    """codes (packed), scales (padded to 4 a row) and the values they stand for, in 32 bits."""
    rows, k = x.shape
    kp = (k + 31) // 32 * 32
    v = torch.zeros(rows, kp, device=x.device)
    v[:, :k] = x.float()
    v = v.reshape(rows, kp // 32, 32)
    most = v.abs().amax(2)
    e = torch.where(most > 0, torch.frexp(most).exponent - 1 - EMAX[bits], torch.full_like(most, -127, dtype=torch.int32)).clamp(-127, 127)
    u = v * _two(-e[..., None])
    if bits == 4:
        a = u.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        q = (torch.round(a / step) * step).clamp(max=6)
        code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)    # 0 .5 1 1.5 2 3 4 6
        code = code | ((u < 0) & (q > 0)).to(torch.uint8) << 3
        code = code.reshape(rows, kp // 2, 2)
        codes = code[..., 0] | code[..., 1] << 4
        q = torch.where(u < 0, -q, q)
    else:
        f = u.clamp(-448, 448).to(torch.float8_e4m3fn)
        codes = f.view(torch.uint8).reshape(rows, kp)
        q = f.float()
    scales = torch.zeros(rows, (kp // 32 + 3) // 4 * 4, dtype=torch.uint8, device=x.device)
    scales[:, :kp // 32] = (e + 127).to(torch.uint8)
    return codes, scales, (q * _two(e[..., None])).reshape(rows, kp)[:, :k]


def _values(codes, scales, bits, k):
    rows = codes.shape[0]
    if bits == 4:
        c = torch.stack((codes & 15, codes >> 4), 2).reshape(rows, -1)
        q = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)[c.long()]
    else:
        q = codes.view(torch.float8_e4m3fn).float()
    q = q.reshape(rows, -1, 32)
    return (q * _two(scales[:, :q.shape[1], None].int() - 127)).reshape(rows, -1)[:, :k]


# ---- plain forms ----

def _places(off, rows):
    """Map and place in the map of each packed row."""
    at = torch.arange(rows, device=off.device, dtype=torch.int32)
    g = (at[:, None] >= off[None, 1:]).sum(1)
    return g, at - off[g]


def _padded(x, g, at, groups, most):
    p = torch.zeros(groups, most, x.shape[1], device=x.device)
    p[g, at] = x.float()
    return p


def _plain(s):
    c, t = s["case"], s["type"]
    op = c["op"]
    if op in ("grouped", "grouped_train"):
        g, at = _places(s["off"], c["rows"])
        x, w = _padded(s["x"], g, at, c["groups"], s["most"]), s["w"].float()
        y = torch.matmul(x, w.transpose(1, 2))[g, at].to(t)
        if op == "grouped":
            return y
        dy = _padded(s["dy"], g, at, c["groups"], s["most"])
        return {"y": y, "dx": torch.matmul(dy, w)[g, at].to(t), "dw": torch.matmul(dy.transpose(1, 2), x).to(t)}
    if op in ("norm", "norm_train"):
        h = s["x"].float() + s["r"].float()
        rstd = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
        y = h * rstd * s["gain"]
        out = {"h": h.to(t), "values": _quantise(y, 8)[2].to(torch.bfloat16)}
        if op == "norm_train":
            dy = s["dy"].float()
            u, n = dy * s["gain"], h * rstd
            out["dx"] = (rstd * (u - n * (u * n).mean(1, keepdim=True)) + s["dh"].float()).to(t)
            out["dgain"] = (dy * n).sum(0)
        return out
    if op == "quantise":
        return _quantise(s["x"], c["bits"])[2].to(torch.bfloat16)
    x = _quantise(s["x"], c["bits"])[2]
    b = _values(s["codes"].flatten(0, 1), s["scales"].flatten(0, 1), c["bits"], c["k"]).reshape(c["groups"], c["n"], c["k"])
    if c["groups"] == 1:
        return torch.matmul(x, b[0].T).to(torch.float16)
    g, at = _places(s["off"], c["rows"])
    return torch.matmul(_padded(x, g, at, c["groups"], s["most"]), b.transpose(1, 2))[g, at].to(torch.float16)


# ---- the framework's calls ----

_module = None


def _products():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "robot-agent_b200"))
        from scenemap_b200 import products
        _module = products
    return _module


def _own(s):
    P = _products()
    c = s["case"]
    op = c["op"]
    if op == "grouped":
        return P.grouped(s["x"], s["w"], s["off"])
    if op == "grouped_train":
        return {"y": P.grouped(s["x"], s["w"], s["off"]), "dx": P.grouped_dx(s["dy"], s["w"], s["off"]), "dw": P.grouped_dw(s["dy"], s["x"], s["off"])}
    if op in ("norm", "norm_train"):
        f = P.norm_add(s["x"], s["r"], s["gain"], eps=EPS, bits=8, values=True)
        out = {"h": f.h, "values": f.values}
        if op == "norm_train":
            out["dx"], out["dgain"] = P.norm_add_backward(s["dy"], f, s["gain"], dh=s["dh"])
        return out
    if op == "quantise":
        return P.mx_quantise(s["x"], c["bits"], values=True).values
    x = P.mx_quantise(s["x"], c["bits"])
    bank = P.MxRows(s["codes"], s["scales"], c["bits"], c["k"])
    return P.mx_product(x, bank, None if c["groups"] == 1 else s["off"], out_dtype=torch.float16)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op, rows, k = case["op"], case["rows"], case["k"]
    b = SIZE[case["type"]]
    blocks = (k + 31) // 32
    if op in ("norm", "norm_train"):
        io = rows * (k * (3 * b + 1 + 2) + blocks) + 4 * k          # x, residual, sum; codes, values, scales
        fl = 8 * rows * k
        if op == "norm_train":                                       # dy, dh, dx, dgain
            io += rows * k * 3 * b + 4 * k
            fl += 12 * rows * k
        return {"bytes": io, "flops": fl}
    if op == "quantise":
        return {"bytes": rows * (k * b + k * 2 + blocks * (32 * case["bits"] // 8 + 1)), "flops": 4 * rows * k}
    g, n = case["groups"], case["n"]
    used = g - case["empty"]
    if op == "grouped":
        return {"bytes": b * (rows * (k + n) + used * n * k), "flops": 2 * rows * n * k}
    if op == "grouped_train":
        return {"bytes": b * (rows * (2 * k + 2 * n) + (used + g) * n * k), "flops": 6 * rows * n * k}
    row = blocks * (32 * case["bits"] // 8 + 1)
    return {"bytes": rows * (k * b + row + 2 * n) + used * n * row, "flops": 2 * rows * n * k}


# ---- the definitions in 64 bits, map by map ----

def _grid(bits):
    if bits == 4:
        pos = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    else:
        pos = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    return torch.tensor(pos, dtype=torch.float64, device="cuda")


def _nearest(y, bits):
    """Each block of 32 over 2^(floor(log2 of its largest) - emax), to the nearest value of the
    format (half-way: the one of even index, which has the even mantissa), times that power."""
    rows, k = y.shape
    pos = _grid(bits)
    v = torch.nn.functional.pad(y, (0, -k % 32)).reshape(rows, -1, 32)
    most = v.abs().amax(2, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent.double() - 1 - EMAX[bits], torch.full_like(most, -127.0)).clamp(-127, 127)
    two = _two(e).double()
    u = v / two
    a = u.abs().contiguous()
    hi = torch.searchsorted(pos, a).clamp(1, len(pos) - 1)
    lo = hi - 1
    up = a - pos[lo] > pos[hi] - a
    tie = a - pos[lo] == pos[hi] - a
    i = torch.where(up | (tie & (hi % 2 == 0)), hi, lo)
    return (torch.sign(u) * pos[i] * two).reshape(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm_train"):
        h = s["x"].double() + s["r"].double()
        n = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["k"] + EPS)
        gain = s["gain"].double()
        out = {"h": h, "values": _nearest(n * gain, 8)}
        if op == "norm_train":
            u = s["dy"].double() * gain
            inv = 1 / torch.sqrt((h * h).sum(1, keepdim=True) / case["k"] + EPS)
            out["dx"] = inv * u - inv * n * ((u * n).sum(1, keepdim=True) / case["k"]) + s["dh"].double()
            out["dgain"] = (s["dy"].double() * n).sum(0)
        return out
    if op == "quantise":
        return _nearest(s["x"].double(), case["bits"])
    off = s["off"].tolist()
    spans = [(g, slice(off[g], off[g + 1])) for g in range(case["groups"])]
    if op == "scores":
        x = _nearest(s["x"].double(), case["bits"])
        y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for g, r in spans:
            pos = torch.cat((_grid(case["bits"]), -_grid(case["bits"])))
            if case["bits"] == 4:
                at = torch.stack((s["codes"][g] % 16, s["codes"][g] // 16), 2).flatten(1).long()
            else:
                code = s["codes"][g].long()
                at = torch.where(code >= 128, code - 128 + len(pos) // 2, code)
            q = pos[at].reshape(case["n"], -1, 32)
            b = q * _two(s["scales"][g][:, :q.shape[1], None].int() - 127).double()
            y[r] = x[r] @ b.reshape(case["n"], -1)[:, :case["k"]].T
        return y
    y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    dx = torch.empty(case["rows"], case["k"], dtype=torch.float64, device="cuda")
    dw = torch.empty(case["groups"], case["n"], case["k"], dtype=torch.float64, device="cuda") if op == "grouped_train" else None
    for g, r in spans:
        w = s["w"][g].double()
        y[r] = s["x"][r].double() @ w.T
        if dw is not None:
            dx[r] = s["dy"][r].double() @ w
            dw[g] = s["dy"][r].double().T @ s["x"][r].double()
    return y if dw is None else {"y": y, "dx": dx, "dw": dw}
