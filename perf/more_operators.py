"""Work of the norm, microscaled and routed-layer operators, as measurable cases.

A layer adds its input to the residual stream, takes the RMS norm, and hands its products rows of
8 bits with scales; training also runs the norm's gradient.  A microscaled linear quantizes each
token to E2M1 or E4M3 with a power-of-two scale for every 32 elements and multiplies with a
weight of E2M1 kept the same way.  A routed layer of a few tokens runs gate, up, down and the
weighted sum over int8 experts.

Shapes are those of a 12B-class decoder layer (hidden 5120, 8 key/value heads of 128, ffn 14336)
and of a 64-expert layer (hidden 2048, expert ffn 1408), and ranges around them.  An int8 row is
padded with zeros to a multiple of 128 bytes, a microscaled one to 256 elements and its scales to 16
bytes; of two E2M1 codes in a byte the first is in the low bits.

With ``own`` false every pass is elementary torch operations in 32 bits, in 64 where a code hangs
on them: the mean of a norm, whole sums past 2^24, and the gate.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: type ids of include/tiermm.h
IDS = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
#: microscaled formats: id, bits, exponent of the largest number, least exponent, mantissa bits, largest number
MX = {"e2m1": (4, 4, 2, 0, 1, 6.0), "e4m3": (8, 8, 8, -6, 3, 448.0)}
EPS = float(np.float32(1e-5))


def row_bytes(K):
    return -(-K // 128) * 128


def mx_row_bytes(fmt, K):
    return -(-K // 256) * 32 * MX[fmt][1]


def mx_scale_bytes(K):
    return -(-K // 512) * 16


# -------------------------------------------------------------------- cases
def listed():
    moe = {"kind": "moe", "E": 64, "topk": 8, "K": 2048, "F": 1408}
    return [
        # in front of the routed layer of a batched decode step: rows for the router and codes for the experts
        {"name": "norm_decode", "kind": "norm", "M": 8, "K": 5120, "type": "f32", "res": True, "out": "both"},
        # a packed batch in front of its int8 products, and a shorter one in front of microscaled ones
        {"name": "norm_batch", "kind": "norm", "M": 4096, "K": 5120, "type": "bf16", "res": True, "out": "i8"},
        {"name": "norm_e4m3", "kind": "norm", "M": 512, "K": 5120, "type": "bf16", "res": True, "out": "e4m3"},
        # the batch's way back, with the gradient that comes down the residual stream
        {"name": "norm_grad_batch", "kind": "norm_grad", "M": 4096, "K": 5120, "type": "bf16", "res": True},
        # the smallest linear of a decode step, and the largest of a layer
        {"name": "mx_k_proj", "kind": "mx", "M": 1, "N": 1024, "K": 5120, "type": "f32", "x": "e4m3", "bias": True},
        {"name": "mx_gate", "kind": "mx", "M": 1, "N": 14336, "K": 5120, "type": "bf16", "x": "e2m1", "bias": False},
        # a short question against one large projection
        {"name": "mx_prompt", "kind": "mx", "M": 37, "N": 14336, "K": 5120, "type": "f32", "x": "e4m3", "bias": False},
        # a full batch, both formats of x (the largest calls)
        {"name": "mx_batch", "kind": "mx", "M": 4096, "N": 14336, "K": 5120, "type": "bf16", "x": "e2m1", "bias": False},
        {"name": "mx_batch_e4m3", "kind": "mx", "M": 4096, "N": 14336, "K": 5120, "type": "bf16", "x": "e4m3",
         "bias": False},
        # the routed layer of one token, of a batched decode step, and of a few tokens with padding among them
        {"name": "moe_one", "T": 1, "type": "f32", "drop": 0.0, **moe},
        {"name": "moe_decode", "T": 8, "type": "f32", "drop": 0.0, **moe},
        {"name": "moe_few", "T": 64, "type": "bf16", "drop": 0.06, **moe},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "norm_grad", "mx", "mx", "mx", "moe", "moe"))
    c = {"kind": kind, "type": rng.choice(("f32", "f16", "bf16"))}
    if kind in ("norm", "norm_grad"):
        c["M"] = _log(rng, 1, 4096)
        c["K"] = _log(rng, 512, 14336)
        if rng.random() < 0.5:  # most models' sizes are whole tiles
            c["K"] = -(-c["K"] // 128) * 128
        c["res"] = rng.random() < 0.7
        if kind == "norm":
            c["out"] = rng.choice(("y", "i8", "both", "e4m3"))
        while c["M"] * c["K"] > 4096 * 5120:
            c["M"] = c["M"] * 3 // 4
        return c
    if kind == "mx":
        c["M"] = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
        c["N"] = _log(rng, 256, 28672)
        c["K"] = _log(rng, 512, 14336)
        if rng.random() < 0.5:
            c["N"], c["K"] = -(-c["N"] // 128) * 128, -(-c["K"] // 128) * 128
        c["x"] = rng.choice(("e2m1", "e4m3"))
        c["bias"] = rng.random() < 0.3
        while 2.0 * c["M"] * c["N"] * c["K"] > 6.0e11:
            c["M"] = c["M"] * 3 // 4
        return c
    c["T"] = _log(rng, 1, 64)
    c["E"] = rng.choice((8, 16, 40, 64, 128))
    c["topk"] = rng.choice((1, 2, 4, 6, 8))
    c["K"] = _log(rng, 512, 5120)
    c["F"] = _log(rng, 256, 14336)
    if rng.random() < 0.6:
        c["K"], c["F"] = -(-c["K"] // 128) * 128, -(-c["F"] // 64) * 64
    while c["E"] * c["K"] * c["F"] > 64 * 1408 * 2048 * 2:
        c["F"] = c["F"] * 3 // 4
    c["drop"] = rng.choice((0.0, 0.0, 0.06, 0.5))
    return c


# ------------------------------------------------------------------- inputs
class State:
    """What the program holds: tensors and raw addresses."""


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _zeros(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device=DEV)


def _x(g, rows, K, dtype):
    """Activations ~N(0, 1) with one channel in 64 eight times as large."""
    x = torch.randn((rows, K), generator=g, device=DEV)
    x[:, 5::64] *= 8.0
    return x.to(dtype)


def _weight(g, rows, K):
    """int8 rows [rows][row_bytes(K)] as quantized normal rows spread them, and their scales."""
    w = _zeros((rows, row_bytes(K)), torch.int8)
    step = max(1, (1 << 26) // K)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        w[r:r + n, :K] = torch.randn((n, K), generator=g, device=DEV).mul_(32.0).round_().clamp_(-127, 127)
    return w, torch.rand(rows, generator=g, device=DEV).mul_(0.4).add_(0.8).mul_(0.02 / 32)


def _mx_weight(g, rows, K):
    """E2M1 rows and their scales of a normal weight of 0.02."""
    w = _zeros((rows, mx_row_bytes("e2m1", K)), torch.uint8)
    s = _zeros((rows, mx_scale_bytes(K)), torch.uint8)
    blocks, levels = -(-K // 32), torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    step = max(1, (1 << 25) // K)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        v, b = _mx(torch.randn((n, K), generator=g, device=DEV).mul_(0.02), "e2m1")
        code = torch.bucketize(v.abs(), levels) + 8 * (v < 0)
        code = torch.nn.functional.pad(code, (0, K % 2)).view(n, -1, 2)
        w[r:r + n, :(K + 1) // 2] = (code[..., 0] + 16 * code[..., 1]).to(torch.uint8)
        s[r:r + n, :blocks] = b.to(torch.uint8)
    return w, s


def _route(c, g):
    """Router choices of T tokens: ids [T][topk] (-1 for a dropped pair) and weights [T][topk]."""
    p = torch.softmax(torch.randn((c["T"], c["E"]), generator=g, device=DEV), -1)
    w, e = torch.topk(p, c["topk"], -1)
    e = e.to(torch.int32)
    out = torch.rand((c["T"], 1 if c["drop"] < 0.1 else c["topk"]), generator=g, device=DEV) < c["drop"]
    return torch.where(out, -1, e).contiguous(), (w / w.sum(-1, keepdim=True)).contiguous()


def _operands(case, seed):
    """The inputs of a case, the same for prepare and exact."""
    c, g, kind = case, _gen(seed), case["kind"]
    dt = TYPES[c["type"]]
    s = State()
    s.case = c
    if kind == "mx":
        s.x = _x(g, c["M"], c["K"], dt)
        s.w, s.sw = _mx_weight(g, c["N"], c["K"])
        s.bias = torch.randn(c["N"], generator=g, device=DEV) if c["bias"] else None
        return s
    if kind == "moe":
        E, K, F = c["E"], c["K"], c["F"]
        s.ids, s.weights = _route(c, g)
        x = _x(g, c["T"], K, torch.float32)
        s.sx = x.abs().amax(1) / 127.0
        s.x = _zeros((c["T"], row_bytes(K)), torch.int8)
        s.x[:, :K] = (x / s.sx[:, None]).round_()
        s.wg, s.sg = _weight(g, E * 2 * F, K)
        s.wd, s.sd = _weight(g, E * K, F)
        flat = s.ids.reshape(-1)
        s.most = max(1, int(torch.bincount(flat[flat >= 0].long(), minlength=1).max())) if bool((flat >= 0).any()) else 1
        return s
    M, K = c["M"], c["K"]
    s.x = _x(g, M, K, dt)
    s.gain = torch.randn(K, generator=g, device=DEV).mul_(0.1).add_(1.0)
    s.res = torch.randn((M, K), generator=g, device=DEV).mul_(2.0).to(dt) if c["res"] else None
    if kind == "norm_grad":  # the rows that the norm saw, its own factor of each, and what comes back
        s.rstd = (1.0 / (s.x.double().square().mean(1) + EPS).sqrt()).float()
        s.dy = torch.randn((M, K), generator=g, device=DEV).mul_(0.1).to(dt)
    return s


def _at(t):
    return None if t is None else t.data_ptr()


def prepare(case, seed):
    s, c, kind = _operands(case, seed), case, case["kind"]
    t, dt, f32 = IDS[c["type"]], TYPES[c["type"]], torch.float32
    K = c["K"]
    if kind == "mx":
        M, N = c["M"], c["N"]
        s.y = _zeros((M, N), dt)
        s.args = (_at(s.x), t, K, MX[c["x"]][0], _at(s.w), mx_row_bytes("e2m1", K), _at(s.sw), mx_scale_bytes(K),
                  _at(s.bias), _at(s.y), t, N, M, N, K)
        return s
    if kind == "moe":
        T, E, F = c["T"], c["E"], c["F"]
        s.y = _zeros((T, K), dt)
        s.args = (_at(s.x), row_bytes(K), _at(s.sx), _at(s.ids), _at(s.weights), _at(s.wg), row_bytes(K), _at(s.sg),
                  _at(s.wd), row_bytes(F), _at(s.sd), _at(s.y), t, K, T, c["topk"], E, K, F)
        return s
    M = c["M"]
    if kind == "norm_grad":
        s.dx, s.dgain = _zeros((M, K), dt), _zeros(K, f32)
        s.args = (_at(s.dy), t, K, _at(s.x), K, _at(s.gain), _at(s.rstd), _at(s.res), K, _at(s.dx), K, _at(s.dgain),
                  M, K)
        return s
    out = c["out"]
    s.h = _zeros((M, K), dt) if c["res"] else None
    s.y = _zeros((M, K), dt) if out in ("y", "both") else None
    head = (_at(s.x), t, K, _at(s.res), K, _at(s.gain), EPS, _at(s.h), K, _at(s.y), K)
    if out == "e4m3":
        rb, sb = mx_row_bytes(out, K), mx_scale_bytes(K)
        s.q, s.scale = _zeros((M, rb), torch.uint8), _zeros((M, sb), torch.uint8)
        s.args = head + (MX[out][0], _at(s.q), rb, _at(s.scale), sb, None, M, K)
    else:
        s.q = _zeros((M, row_bytes(K)), torch.int8) if out != "y" else None
        s.scale = _zeros(M, f32) if out != "y" else None
        s.args = head + (_at(s.q), row_bytes(K), _at(s.scale), None, M, K)
    return s


# -------------------------------------------------------------- plain forms
def _mx(y, fmt):
    """Elements of fp32 rows as the format holds them, under the scale of their 32, and the scales' bytes."""
    _, _, emax, emin, bits, most = MX[fmt]
    M, K = y.shape
    b = torch.nn.functional.pad(y, (0, -K % 32)).view(M, -1, 32)
    top = b.abs().amax(-1)
    byte = torch.where(top > 0, (torch.frexp(top)[1] - 1 - emax + 127).clamp(0, 254), 0)
    v = torch.ldexp(b, 127 - byte[..., None])
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=emin).float() - bits)
    v = ((v / step).round() * step).clamp(-most, most)
    return v.view(M, -1)[:, :K], byte


def _mx_values(v, byte):
    """The numbers that elements and scales stand for."""
    M, K = v.shape
    s = torch.exp2(byte.float() - 127.0)
    return v * s[:, :-(-K // 32)].repeat_interleave(32, 1)[:, :K]


def _mx_weight_values(s, K):
    """The numbers of an E2M1 weight."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    levels = torch.cat([levels, -levels])
    code = torch.stack([s.w & 15, s.w >> 4], -1).view(s.w.shape[0], -1)[:, :K]
    return _mx_values(levels[code.long()], s.sw)


def _codes(v):
    """Whole numbers -127..127 and the scale of each row."""
    top = v.abs().amax(1)
    steps = torch.full_like(top, 127.0)
    inverse = torch.where(top > 0, steps / top, torch.zeros_like(top))
    return (v * inverse[:, None]).round(), top / steps


def _plain_moe(s):
    c, E, K, F, k = s.case, s.case["E"], s.case["K"], s.case["F"], s.case["topk"]
    T, P = c["T"], c["T"] * c["topk"]
    # every expert's pairs padded to the fullest one's, batched products of whole numbers in 64 bits
    flat = s.ids.reshape(-1)
    key = torch.where((flat < 0) | (flat >= E), E, flat).long()
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(E, device=DEV)).sum(0)
    first = torch.cumsum(counts, 0) - counts
    place = first[:, None] + torch.arange(s.most, device=DEV)
    inside = place < (first + counts)[:, None]
    pair = torch.where(inside, order[place.clamp(max=P - 1)], 0)
    token = torch.div(pair, k, rounding_mode="floor")
    x, sx = s.x[token][..., :K].double(), s.sx[token][..., None]
    wg = s.wg[:, :K].view(E, 2 * F, K).transpose(1, 2).double().contiguous()
    gu = torch.bmm(x, wg).float() * (sx * s.sg.view(E, 1, 2 * F))
    g, u = gu[..., :F].double(), gu[..., F:].double()
    h = (g / (1.0 + torch.exp(-g)) * u).float()
    q, sh = _codes(h.view(-1, F))
    wd = s.wd[:, :F].view(E, K, F).transpose(1, 2).double().contiguous()
    y = torch.bmm(q.view(E, -1, F).double(), wd).float() * (sh.view(E, -1, 1) * s.sd.view(E, 1, K))
    # back to the tokens: each pair's row, zeros for a dropped one
    rank = torch.empty_like(order)
    rank[order] = torch.arange(P, device=DEV)
    e = key.clamp(max=E - 1)
    got = y[e, (rank - first[e]).clamp(0, s.most - 1)] * s.weights.reshape(-1)[:, None]
    got = torch.where((key < E)[:, None], got, torch.zeros((), device=DEV))
    return got.view(T, k, K).sum(1).to(TYPES[c["type"]])


def _plain(s):
    c, kind = s.case, s.case["kind"]
    dt, K = TYPES[c["type"]], c["K"]
    if kind == "mx":
        y = _mx_values(*_mx(s.x.float(), c["x"])) @ _mx_weight_values(s, K).t()
        return (y + s.bias if c["bias"] else y).to(dt)
    if kind == "moe":
        return _plain_moe(s)
    if kind == "norm_grad":
        xh = s.x.float() * s.rstd[:, None]
        dy = s.dy.float()
        d = dy * s.gain
        dx = (d - xh * (d * xh).mean(1, keepdim=True)) * s.rstd[:, None]
        return {"dx": (dx + s.res.float() if c["res"] else dx).to(dt), "dgain": (dy * xh).sum(0)}
    h = (s.x.float() + s.res.float()).to(dt) if c["res"] else s.x
    rstd = (1.0 / (h.double().square().mean(1) + EPS).sqrt()).float()
    y = (h.float() * rstd[:, None]) * s.gain
    got = {"h": h if c["res"] else None, "y": y.to(dt) if c["out"] in ("y", "both") else None}
    if c["out"] == "e4m3":
        v, byte = _mx(y, "e4m3")
        return {**got, "q": v.to(torch.float8_e4m3fn), "scale": byte.to(torch.uint8)}
    if c["out"] != "y":
        q, scale = _codes(y)
        got = {**got, "q": q.to(torch.int8), "scale": scale}
    return got


# --------------------------------------------------------------------- pass
def run(s):
    if not own:
        return _plain(s)
    import tier_amd

    c, kind = s.case, s.case["kind"]
    if kind == "mx":
        tier_amd.mx_linear(*s.args)
        return s.y
    if kind == "moe":
        tier_amd.moe_i8_layer(*s.args)
        return s.y
    if kind == "norm_grad":
        tier_amd.rms_norm_grad(*s.args)
        return {"dx": s.dx, "dgain": s.dgain}
    K = c["K"]
    got = {"h": s.h, "y": s.y}
    if c["out"] == "e4m3":  # an element's 8 bits are a number of torch's own type
        tier_amd.rms_norm_mx(*s.args)
        return {**got, "q": s.q.view(torch.float8_e4m3fn)[:, :K], "scale": s.scale[:, :-(-K // 32)]}
    tier_amd.rms_norm(*s.args)
    if c["out"] != "y":  # whole numbers, fixed by the 32-bit steps behind the mean
        got = {**got, "q": s.q[:, :K], "scale": s.scale}
    return got


def work(case):
    c, kind = case, case["kind"]
    es, K = SIZE[c["type"]], c["K"]
    if kind == "mx":
        M, N = c["M"], c["N"]
        return {"bytes": N * (K / 2 + K / 32) + (4 * N if c["bias"] else 0) + es * M * (K + N), "flops": 2 * M * N * K}
    if kind == "moe":
        T, E, k, F = c["T"], c["E"], c["topk"], c["F"]
        # experts that some token takes, as independent draws of topk of E
        used = E * (1 - (1 - k / E * (1 - c["drop"])) ** T)
        return {"bytes": used * (3 * F * K + 8 * F + 4 * K) + 8 * T * k + T * K * (1 + es),
                "flops": 6 * T * k * (1 - c["drop"]) * F * K}
    M, res = c["M"], c["res"]
    if kind == "norm_grad":
        return {"bytes": es * M * K * (4 if res else 3) + 8 * K + 4 * M, "flops": 8 * M * K}
    out = {"y": es, "i8": 1, "both": es + 1, "e4m3": 1 + 1 / 32}[c["out"]]
    return {"bytes": M * K * (es * (3 if res else 1) + out) + 4 * K + 4 * M, "flops": 6 * M * K}


# ------------------------------------------------------------------ 64 bits
def _nearest64(v, fmt):
    """v on the format's numbers, by a search among them: ties to the even code."""
    if fmt == "e2m1":
        levels = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        levels = [m / 8 * 2.0 ** -6 for m in range(8)]
        levels += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if e < 8 or m < 7]
    n = torch.tensor(levels, dtype=torch.float64, device=DEV)
    a = v.abs().clamp(max=levels[-1])
    hi = torch.searchsorted(n, a).clamp(max=len(levels) - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = a - n[lo], n[hi] - a
    take = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return n[take] * v.sign()


def _mx64(y, fmt):
    """Rows of 64-bit numbers as the format and its scales hold them: elements, and scales of 32."""
    M, K = y.shape
    b = torch.cat([y, torch.zeros((M, -K % 32), dtype=torch.float64, device=DEV)], 1).view(M, -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))  # (exact at powers of two)
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e)) - MX[fmt][2]
    s = torch.exp2(e.clamp(min=-127.0, max=127.0))
    return _nearest64(b / s, fmt), s


def _exact_moe(s):
    c, E, K, F, k = s.case, s.case["E"], s.case["K"], s.case["F"], s.case["topk"]
    out = torch.zeros((c["T"], K), dtype=torch.float64, device=DEV)
    ids, x, one = s.ids.long(), s.x[:, :K].double(), np.float32(127)
    for e in ids[(ids >= 0) & (ids < E)].unique().tolist():
        t, j = (ids == e).nonzero(as_tuple=True)
        wg = s.wg[2 * F * e:2 * F * (e + 1), :K].double()
        gu = (x[t] @ wg.t().contiguous()).cpu().numpy().astype(np.float32)
        gu = gu * (s.sx[t, None] * s.sg[2 * F * e:2 * F * (e + 1)]).cpu().numpy()
        g, u = gu[:, :F].astype(np.float64), gu[:, F:].astype(np.float64)
        # h's whole numbers are defined by 32-bit steps, as the int8 rows of any other product
        h = (u * g / (np.exp(-g) + 1.0)).astype(np.float32)
        top = abs(h).max(1, keepdims=True)
        inverse = np.where(top > 0, one / np.maximum(top, np.float32(1e-30)), np.float32(0))
        q = torch.from_numpy((h * inverse).round().astype(np.float64)).to(DEV)
        wd = s.wd[K * e:K * (e + 1), :F].double()
        y = (q @ wd.t().contiguous()) * torch.from_numpy(top.astype(np.float64) / 127).to(DEV)
        out.index_put_((t,), y * s.sd[K * e:K * (e + 1)].double() * s.weights[t, j].double()[:, None], accumulate=True)
    return out


def exact(case, seed):
    s, c, kind = _operands(case, seed), case, case["kind"]
    K = c["K"]
    if kind == "mx":
        v, sc = _mx64(s.x.double(), c["x"])
        x = (v * sc).view(c["M"], -1)[:, :K]
        w = torch.zeros((c["N"], K), dtype=torch.float64, device=DEV)
        n = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.float64, device=DEV) / 2
        w[:, 0::2] = n[(s.w % 16).long()][:, :(K + 1) // 2]
        w[:, 1::2] = n[torch.div(s.w, 16, rounding_mode="floor").long()][:, :K // 2]
        at = torch.div(torch.arange(K, device=DEV), 32, rounding_mode="floor")
        w *= torch.pow(2.0, s.sw.double() - 127)[:, at]
        y = x @ w.t().contiguous()
        return y + s.bias.double() if c["bias"] else y
    if kind == "moe":
        return _exact_moe(s)
    if kind == "norm_grad":
        r, g = s.rstd.double()[:, None], s.gain.double()
        x, dy = s.x.double(), s.dy.double()
        dot = (dy * g * x).sum(1, keepdim=True)
        dx = r * dy * g - x * dot * r ** 3 / K
        return {"dx": dx + s.res.double() if c["res"] else dx, "dgain": (dy * (x * r)).sum(0)}
    dt = TYPES[c["type"]]
    whole = s.x.double() + s.res.double() if c["res"] else s.x.double()
    h = whole.to(dt).double() if c["type"] != "f32" else whole.float().double()
    y = h / (h.pow(2).sum(1, keepdim=True) / K + EPS).sqrt() * s.gain.double()
    got = {"h": whole if c["res"] else None, "y": y if c["out"] in ("y", "both") else None}
    if c["out"] == "e4m3":
        return {**got, "q": _mx64(y, "e4m3")[0].view(c["M"], -1)[:, :K], "scale": None}
    if c["out"] != "y":
        got = {**got, "q": None, "scale": y.abs().amax(1) / 127}
    return got
