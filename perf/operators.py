"""Work of the routed-token and int8 operators, as measurable cases.

A routed layer sorts its tokens by expert, multiplies each expert's rows, and brings them
back weighted; training also runs both ways' gradients.  An int8 linear quantizes each
token (a scale per row) and multiplies with a weight kept in int8 with a scale per output
channel; the experts' form reads its rows through the sorted pairs.

Shapes are those of a 12B-class decoder layer (hidden 5120, 8 key/value heads of 128, ffn
14336) and of a 64-expert layer (hidden 2048, expert ffn 1408, gate and up stacked), and
ranges around them.  An int8 row is padded with zeros to a multiple of 128 bytes.

With ``own`` false every pass is elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: type ids of include/tiermm.h
IDS = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def row_bytes(K):
    return -(-K // 128) * 128


# -------------------------------------------------------------------- cases
def listed():
    moe = {"E": 64, "topk": 8, "K": 2048}
    return [
        # the eight tokens of a batched decode step on their way to the experts and back
        {"name": "sort_decode", "kind": "sort", "T": 8, "type": "f32", "drop": 0.0, **moe},
        {"name": "unsort_decode", "kind": "unsort", "T": 8, "type": "f32", "drop": 0.0, **moe},
        # a packed training batch, both ways and both gradients; in bf16 with padding tokens unrouted
        {"name": "sort_batch", "kind": "sort", "T": 4096, "type": "f32", "drop": 0.0, **moe},
        {"name": "sort_grad_batch", "kind": "sort_grad", "T": 4096, "type": "bf16", "drop": 0.06, **moe},
        {"name": "unsort_batch", "kind": "unsort", "T": 4096, "type": "bf16", "drop": 0.06, **moe},
        {"name": "unsort_grad_batch", "kind": "unsort_grad", "T": 4096, "type": "f32", "drop": 0.0, **moe},
        # the smallest linear of a decode step: the k projection of one token
        {"name": "i8_k_proj", "kind": "i8", "M": 1, "N": 1024, "K": 5120, "type": "f32", "bias": True},
        # the largest one of a layer
        {"name": "i8_gate", "kind": "i8", "M": 1, "N": 14336, "K": 5120, "type": "bf16", "bias": False},
        # a short question against one large projection
        {"name": "i8_prompt", "kind": "i8", "M": 37, "N": 14336, "K": 5120, "type": "f32", "bias": False},
        # a full batch (the largest call)
        {"name": "i8_batch", "kind": "i8", "M": 4096, "N": 14336, "K": 5120, "type": "bf16", "bias": False},
        # gate and up of the routed experts, for the eight tokens and for the batch
        {"name": "experts_decode", "kind": "experts", "T": 8, "N": 2816, "type": "f32", "drop": 0.0, **moe},
        {"name": "experts_batch", "kind": "experts", "T": 4096, "N": 2816, "type": "bf16", "drop": 0.0, **moe},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("sort", "sort_grad", "unsort", "unsort_grad", "i8", "i8", "i8", "experts", "experts"))
    c = {"kind": kind, "type": rng.choice(("f32", "f16", "bf16"))}
    if kind == "i8":
        c["M"] = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
        c["N"] = _log(rng, 256, 28672)
        c["K"] = _log(rng, 512, 14336)
        if rng.random() < 0.5:  # most models' sizes are whole tiles
            c["N"], c["K"] = -(-c["N"] // 128) * 128, -(-c["K"] // 128) * 128
        c["bias"] = rng.random() < 0.3
        while 2.0 * c["M"] * c["N"] * c["K"] > 6.0e11:
            c["M"] = c["M"] * 3 // 4
        return c
    c["T"] = _log(rng, 1, 4096)
    c["E"] = rng.choice((8, 16, 40, 64, 128))
    c["topk"] = rng.choice((1, 2, 4, 6, 8))
    c["K"] = _log(rng, 512, 5120)
    if rng.random() < 0.6:
        c["K"] = -(-c["K"] // 128) * 128
    c["drop"] = rng.choice((0.0, 0.0, 0.06, 0.5))
    if kind == "experts":
        c["N"] = _log(rng, 256, 2816)
        c["K"] = min(c["K"], 2048)
        if rng.random() < 0.6:
            c["N"] = -(-c["N"] // 64) * 64
    else:
        while c["T"] * c["topk"] * c["K"] > 4096 * 8 * 2048:
            c["T"] = c["T"] * 3 // 4
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
    if kind == "i8":
        s.x = _x(g, c["M"], c["K"], dt)
        s.w, s.sw = _weight(g, c["N"], c["K"])
        s.bias = torch.randn(c["N"], generator=g, device=DEV) if c["bias"] else None
        return s
    T, E, k, K = c["T"], c["E"], c["topk"], c["K"]
    P = T * k
    s.ids, s.weights = _route(c, g)
    if kind == "sort":
        s.x = torch.randn((T, K), generator=g, device=DEV).to(dt)
        return s
    s.offsets, s.pairs, s.sorted = _plan(s.ids, E)
    if kind == "experts":
        s.x = _x(g, T, K, dt)
        s.w, s.sw = _weight(g, E * c["N"], K)
        counts = torch.diff(s.offsets)
        s.most = max(1, int(counts.max()))
        return s
    if kind != "unsort_grad":
        s.x = torch.randn((P, K), generator=g, device=DEV).to(dt)
        return s
    s.x = torch.randn((P, K), generator=g, device=DEV).to(dt)
    s.dout = torch.randn((T, K), generator=g, device=DEV).to(dt)
    return s


def prepare(case, seed):
    s, c, kind = _operands(case, seed), case, case["kind"]
    t, dt, i32 = IDS[c["type"]], TYPES[c["type"]], torch.int32
    if kind == "i8":
        M, N, K = c["M"], c["N"], c["K"]
        s.y = _zeros((M, N), dt)
        s.args = (s.x.data_ptr(), t, K, s.w.data_ptr(), row_bytes(K), s.sw.data_ptr(),
                  s.bias.data_ptr() if c["bias"] else None, s.y.data_ptr(), t, N, M, N, K)
        return s
    T, E, k, K = c["T"], c["E"], c["topk"], c["K"]
    P = T * k
    if kind == "sort":
        s.offsets, s.pairs, s.sorted = _zeros(E + 1, i32), _zeros((T, k), i32), _zeros(P, i32)
        s.y = _zeros((P, K), dt)
        s.plan_args = (s.ids.data_ptr(), T, k, E, s.offsets.data_ptr(), s.pairs.data_ptr(), s.sorted.data_ptr())
        s.args = (s.x.data_ptr(), t, K, s.pairs.data_ptr(), s.sorted.data_ptr(), s.y.data_ptr(), K, T, k, K)
    elif kind == "sort_grad":
        s.y = _zeros((T, K), dt)
        s.args = (s.x.data_ptr(), t, K, s.pairs.data_ptr(), s.y.data_ptr(), K, T, k, K)
    elif kind == "unsort":
        s.y = _zeros((T, K), dt)
        s.args = (s.x.data_ptr(), t, K, s.pairs.data_ptr(), s.weights.data_ptr(), s.y.data_ptr(), K, T, k, K)
    elif kind == "unsort_grad":
        s.y, s.dw = _zeros((P, K), dt), _zeros((T, k), torch.float32)
        s.args = (s.dout.data_ptr(), t, K, s.x.data_ptr(), K, s.pairs.data_ptr(), s.sorted.data_ptr(),
                  s.weights.data_ptr(), s.y.data_ptr(), K, s.dw.data_ptr(), T, k, K)
    else:
        N, rb = c["N"], row_bytes(K)
        s.q, s.sx = _zeros((T, rb), torch.int8), _zeros(T, torch.float32)
        s.y = _zeros((P, N), dt)
        s.quant_args = (s.x.data_ptr(), t, K, s.q.data_ptr(), rb, s.sx.data_ptr(), T, K)
        s.args = (s.q.data_ptr(), rb, s.sx.data_ptr(), s.sorted.data_ptr(), T, k, s.offsets.data_ptr(), E,
                  s.w.data_ptr(), rb, s.sw.data_ptr(), s.y.data_ptr(), t, N, P, N, K)
    return s


# -------------------------------------------------------------- plain forms
def _plan(ids, E):
    """Pairs sorted by expert, in order within one: offsets [E + 1], places [T][topk], pairs [P]."""
    flat = ids.reshape(-1)
    dropped = (flat < 0) | (flat >= E)
    key = torch.where(dropped, E, flat)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel(), device=DEV)
    counts = (key[:, None] == torch.arange(E, device=DEV)).sum(0)
    offsets = torch.cat([_zeros(1, torch.int64), torch.cumsum(counts, 0)])
    pairs = torch.where(dropped, -1, place)
    inside = torch.arange(flat.numel(), device=DEV) < offsets[-1]
    return (offsets.to(torch.int32), pairs.to(torch.int32).view(ids.shape),
            torch.where(inside, order, -1).to(torch.int32))


def _rows(x, index):
    """Rows of x in 32 bits, zeros where the index is negative."""
    got = x[index.clamp(min=0).long()].float()
    return torch.where((index >= 0)[..., None], got, torch.zeros((), device=DEV))


def _quant(x):
    """Whole numbers -127..127 and the scale of each row."""
    x = x.float()
    top = x.abs().amax(1)
    steps = torch.full_like(top, 127.0)
    inverse = torch.where(top > 0, steps / top, torch.zeros_like(top))
    return (x * inverse[:, None]).round(), top / steps


def _plain(s):
    c, kind = s.case, s.case["kind"]
    dt, K = TYPES[c["type"]], c["K"]
    if kind == "i8":
        q, sx = _quant(s.x)
        y = (q @ s.w[:, :K].float().t()) * (sx[:, None] * s.sw)
        return (y + s.bias if c["bias"] else y).to(dt)
    k = c["topk"]
    if kind == "sort":
        offsets, pairs, order = _plan(s.ids, c["E"])
        src = torch.where(order >= 0, torch.div(order, k, rounding_mode="floor"), -1)
        return {"offsets": offsets, "pairs": pairs, "sorted": order, "rows": _rows(s.x, src).to(dt)}
    if kind == "sort_grad":
        return _rows(s.x, s.pairs).sum(1).to(dt)
    if kind == "unsort":
        return (_rows(s.x, s.pairs) * s.weights[..., None]).sum(1).to(dt)
    if kind == "unsort_grad":
        src = torch.where(s.sorted >= 0, torch.div(s.sorted, k, rounding_mode="floor"), -1)
        w = s.weights.reshape(-1)[s.sorted.clamp(min=0).long()]
        return {"dy": (_rows(s.dout, src) * w[:, None]).to(dt),
                "dw": (_rows(s.x, s.pairs) * s.dout.float()[:, None]).sum(-1)}
    # experts: every expert's rows padded to the fullest one's, one batched product
    E, N = c["E"], c["N"]
    q, sx = _quant(s.x)
    place = s.offsets[:-1, None] + torch.arange(s.most, device=DEV)
    inside = place < s.offsets[1:, None]
    src = torch.where(inside, torch.div(s.sorted[place.clamp(max=s.sorted.numel() - 1).long()], k,
                                        rounding_mode="floor"), -1)
    w = s.w[:, :K].float().view(E, N, K).transpose(1, 2).contiguous()
    y = torch.bmm(_rows(q, src), w) * s.sw.view(E, 1, N) * _rows(sx[:, None], src)
    p = torch.arange(s.sorted.numel(), device=DEV)
    e = (p[:, None] >= s.offsets[1:]).sum(1)
    got = y[e.clamp(max=E - 1), (p - s.offsets[e.clamp(max=E - 1)]).clamp(max=s.most - 1)]
    return torch.where((e < E)[:, None], got, torch.zeros((), device=DEV)).to(dt)


# --------------------------------------------------------------------- pass
def run(s):
    if not own:
        return _plain(s)
    import tier_amd

    kind = s.case["kind"]
    if kind == "i8":
        tier_amd.i8_linear(*s.args)
        return s.y
    if kind == "sort":
        tier_amd.moe_plan(*s.plan_args)
        tier_amd.moe_sort(*s.args)
        return {"offsets": s.offsets, "pairs": s.pairs, "sorted": s.sorted, "rows": s.y}
    if kind == "sort_grad":
        tier_amd.moe_sort_grad(*s.args)
        return s.y
    if kind == "unsort":
        tier_amd.moe_unsort(*s.args)
        return s.y
    if kind == "unsort_grad":
        tier_amd.moe_unsort_grad(*s.args)
        return {"dy": s.y, "dw": s.dw}
    tier_amd.i8_quant(*s.quant_args)
    tier_amd.i8_gemm_grouped(*s.args)
    return s.y


def work(case):
    c, kind = case, case["kind"]
    es, K = SIZE[c["type"]], c["K"]
    if kind == "i8":
        M, N = c["M"], c["N"]
        return {"bytes": N * K + 4 * N * (2 if c["bias"] else 1) + es * M * (K + N), "flops": 2 * M * N * K}
    T, E, k = c["T"], c["E"], c["topk"]
    P = T * k
    live = P * (1 - c["drop"])
    if kind == "sort":  # every row of the sorted array is written, the unrouted ones as zeros
        return {"bytes": 12 * P + 4 * (E + 1) + es * (T + P) * K, "flops": 0}
    if kind == "sort_grad":
        return {"bytes": 4 * P + es * (live + T) * K, "flops": live * K}
    if kind == "unsort":
        return {"bytes": 8 * P + es * (live + T) * K, "flops": 2 * live * K}
    if kind == "unsort_grad":
        return {"bytes": 16 * P + es * (live + P + T) * K, "flops": 3 * live * K}
    # experts that some token takes, as independent draws of topk of E
    N = c["N"]
    used = E * (1 - (1 - k / E * (1 - c["drop"])) ** T)
    return {"bytes": used * N * (K + 4) + 4 * P + es * (T * K + P * N), "flops": 2 * live * N * K}


# ------------------------------------------------------------------ 64 bits
def _quant64(x):
    """The whole numbers are defined by 32-bit steps: x * fl(127 / max), to nearest even."""
    a = x.float().cpu().numpy()
    top = abs(a).max(1)
    one = top.dtype.type(127)
    inverse = (one / top.clip(min=1e-30)) * (top > 0)
    q = (a * inverse[:, None].astype(a.dtype)).round()
    return torch.from_numpy(q).to(DEV).double(), torch.from_numpy(top).to(DEV).double() / 127


def exact(case, seed):
    s, c, kind = _operands(case, seed), case, case["kind"]
    K = c["K"]
    if kind == "i8":
        q, sx = _quant64(s.x)
        y = (q @ s.w[:, :K].double().t().contiguous()) * sx[:, None] * s.sw.double()
        return y + s.bias.double() if c["bias"] else y
    T, E, k = c["T"], c["E"], c["topk"]
    P = T * k
    if kind == "sort":
        order = sorted((e, i) for i, e in enumerate(s.ids.reshape(-1).tolist()) if 0 <= e < E)
        rows = torch.zeros((P, K), dtype=torch.float64, device=DEV)
        src = torch.tensor([i // k for _, i in order], dtype=torch.int64, device=DEV)
        rows[:len(order)] = s.x.double()[src]
        return {"offsets": None, "pairs": None, "sorted": None, "rows": rows}
    w, pairs = s.weights.double(), s.pairs.long()
    if kind in ("sort_grad", "unsort"):
        out = torch.zeros((T, K), dtype=torch.float64, device=DEV)
        for j in range(k):
            live = pairs[:, j] >= 0
            part = s.x[pairs[live, j]].double()
            out[live] += part if kind == "sort_grad" else part * w[live, j, None]
        return out
    if kind == "unsort_grad":
        dy = torch.zeros((P, K), dtype=torch.float64, device=DEV)
        dw = torch.zeros((T, k), dtype=torch.float64, device=DEV)
        for j in range(k):
            live = pairs[:, j] >= 0
            d = s.dout[live].double()
            dy[pairs[live, j]] = d * w[live, j, None]
            dw[live, j] = (d * s.x[pairs[live, j]].double()).sum(1)
        return {"dy": dy, "dw": dw}
    N, off = c["N"], s.offsets.tolist()
    q, sx = _quant64(s.x)
    y = torch.zeros((P, N), dtype=torch.float64, device=DEV)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        r = torch.div(s.sorted[a:b], k, rounding_mode="floor").long()
        we = s.w[e * N:(e + 1) * N, :K].double().t().contiguous()
        y[a:b] = (q[r] @ we) * sx[r, None] * s.sw[e * N:(e + 1) * N].double()
    return y
