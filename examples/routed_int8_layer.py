"""A routed (mixture of experts) layer on int8 weights, forward and backward to its input.

Tokens choose their experts (softmax, top-k), the plan orders the pairs on the GPU, the
tokens are quantized once and gathered by the experts' products; the weighted sum brings
them back.  Backward runs the same way round: the gradient of the sum, two products on
the transposed weights (laid out once, like the others), the gradient of the sort.  No
host copy of the routing is made, so a captured graph could replay the whole layer.

    python examples/routed_int8_layer.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tier_amd  # noqa: E402

DEV = "cuda"
IDS = {torch.float32: tier_amd.F32, torch.float16: tier_amd.F16, torch.bfloat16: tier_amd.BF16}


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32, device=DEV)


class Int8Weight:
    """Rows [rows][K] of fp32 as int8 codes and a scale each."""

    def __init__(self, w):
        self.rows, self.K = w.shape
        self.rb = tier_amd.i8_row_bytes(self.K)
        self.q = torch.empty((self.rows, self.rb), dtype=torch.int8, device=DEV)
        self.scale = torch.empty(self.rows, device=DEV)
        w = w.contiguous()
        tier_amd.i8_quant(w.data_ptr(), tier_amd.F32, self.K, self.q.data_ptr(), self.rb, self.scale.data_ptr(),
                          self.rows, self.K, stream=_stream())


def _stream():
    return torch.cuda.current_stream().cuda_stream


class RoutedInt8Layer:
    """gate_up [E][2 * ffn][hidden] and down [E][hidden][ffn], fp32 on the GPU."""

    def __init__(self, gate_up, down, topk):
        self.E, f2, self.hidden = gate_up.shape
        self.ffn, self.topk = f2 // 2, topk
        flat = lambda w: Int8Weight(w.reshape(-1, w.shape[-1]))  # noqa: E731
        self.gate_up, self.down = flat(gate_up), flat(down)
        # for the backward pass: the transposed weights, quantized by their own rows
        self.gate_up_t, self.down_t = flat(gate_up.transpose(1, 2)), flat(down.transpose(1, 2))

    def route(self, ids):
        """Plan of ids [T][topk] (int32, anything outside [0, E) is dropped)."""
        T = ids.shape[0]
        self.T, self.P = T, T * self.topk
        self.offsets, self.places, self.sorted = _i32(self.E + 1), _i32(T, self.topk), _i32(self.P)
        n = tier_amd.moe_plan_ws_bytes(T, self.topk, self.E)
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
        tier_amd.moe_plan(ids.data_ptr(), T, self.topk, self.E, self.offsets.data_ptr(), self.places.data_ptr(),
                          self.sorted.data_ptr(), ws.data_ptr() if n else None, n, stream=_stream())

    def _experts(self, x, w, N, gathered):
        """x quantized, times every expert's weight; gathered: rows of x by the sorted pairs."""
        rows, K = x.shape
        q = torch.empty((rows, w.rb), dtype=torch.int8, device=DEV)
        s = torch.empty(rows, device=DEV)
        y = torch.empty((self.P, N), dtype=x.dtype, device=DEV)
        t = IDS[x.dtype]
        tier_amd.i8_quant(x.data_ptr(), t, K, q.data_ptr(), w.rb, s.data_ptr(), rows, K, stream=_stream())
        tier_amd.i8_gemm_grouped(q.data_ptr(), w.rb, s.data_ptr(), self.sorted.data_ptr() if gathered else None, rows,
                                 self.topk, self.offsets.data_ptr(), self.E, w.q.data_ptr(), w.rb, w.scale.data_ptr(),
                                 y.data_ptr(), t, N, self.P, N, K, stream=_stream())
        return y

    def forward(self, x, ids, weights):
        self.route(ids)
        self.weights = weights
        self.gu = self._experts(x, self.gate_up, 2 * self.ffn, True)
        gate, up = self.gu.float().chunk(2, -1)
        self.y = self._experts((torch.nn.functional.silu(gate) * up).to(x.dtype), self.down, self.hidden, False)
        out = torch.empty_like(x)
        tier_amd.moe_unsort(self.y.data_ptr(), IDS[x.dtype], self.hidden, self.places.data_ptr(), weights.data_ptr(),
                            out.data_ptr(), self.hidden, self.T, self.topk, self.hidden, stream=_stream())
        return out

    def backward(self, dout):
        """(dx, dweights) of the last forward; the expert weights are frozen."""
        t, H = IDS[dout.dtype], self.hidden
        dy, dw = torch.empty_like(self.y), torch.empty_like(self.weights)
        tier_amd.moe_unsort_grad(dout.data_ptr(), t, H, self.y.data_ptr(), H, self.places.data_ptr(),
                                 self.sorted.data_ptr(), self.weights.data_ptr(), dy.data_ptr(), H, dw.data_ptr(),
                                 self.T, self.topk, H, stream=_stream())
        dh = self._experts(dy, self.down_t, self.ffn, False).float()
        gate, up = self.gu.float().chunk(2, -1)
        s = torch.sigmoid(gate)
        dgu = torch.cat([dh * up * (s + gate * s * (1 - s)), dh * gate * s], -1).to(dout.dtype)
        dxs = self._experts(dgu, self.gate_up_t, H, False)
        dx = torch.empty_like(dout)
        tier_amd.moe_sort_grad(dxs.data_ptr(), t, H, self.places.data_ptr(), dx.data_ptr(), H, self.T, self.topk, H,
                               stream=_stream())
        return dx, dw


def plain(x, ids, weights, gate_up, down, dout):
    """out, dx, dweights of the same layer on the unquantized weights, in 64 bits (one expert after
    another), and |dout| |y| of every weight: what its gradient, a product of the two, is off by
    goes by their lengths, also where the product itself is next to nothing."""
    x, w, d = x.double(), weights.double(), dout.double()
    out, dx, dw, size = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w)
    for e in range(gate_up.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        gu, dn = gate_up[e].double(), down[e].double()
        g, u = (x[t] @ gu.t().contiguous()).chunk(2, -1)
        s = torch.sigmoid(g)
        y = (g * s * u) @ dn.t().contiguous()
        out.index_add_(0, t, w[t, j, None] * y)
        dw[t, j] = (d[t] * y).sum(-1)
        size[t, j] = d[t].norm(dim=-1) * y.norm(dim=-1)
        dh = (w[t, j, None] * d[t]) @ dn
        dx.index_add_(0, t, torch.cat([dh * u * (s + g * s * (1 - s)), dh * g * s], -1) @ gu)
    return out, dx, dw, size


def example(T=512, E=16, topk=4, hidden=1024, ffn=704, dtype=torch.bfloat16, seed=0):
    """Runs the layer on random weights and tokens (some pairs dropped) and compares it with the
    unquantized one: {name: relative difference}."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    gate_up, down = rand(E, 2 * ffn, hidden) * hidden ** -0.5, rand(E, hidden, ffn) * ffn ** -0.5
    x, dout = rand(T, hidden).to(dtype), rand(T, hidden).to(dtype)
    w, ids = torch.topk(torch.softmax(rand(T, E), -1), topk, -1)
    ids = torch.where(rand(T, topk) > 1.5, -1, ids).to(torch.int32).contiguous()
    w = (w / w.sum(-1, keepdim=True)).contiguous()
    layer = RoutedInt8Layer(gate_up, down, topk)
    out = layer.forward(x, ids, w)
    dx, dw = layer.backward(dout)
    out0, dx0, dw0, size = plain(x, ids, w, gate_up, down, dout)
    off = lambda a, b, by: float((a.double() - b).norm() / by.norm())  # noqa: E731
    return {"out": off(out, out0, out0), "dx": off(dx, dx0, dx0), "dweights": off(dw, dw0, size)}


if __name__ == "__main__":
    tier_amd.init(0)
    for size in ({"T": 1, "E": 8, "topk": 2, "hidden": 256, "ffn": 192},  # one token, few experts
                 {"T": 33, "E": 5, "topk": 3, "hidden": 515, "ffn": 130},  # odd sizes
                 {"T": 700, "E": 16, "topk": 4, "hidden": 1024, "ffn": 704}):
        for dtype in (torch.float32, torch.bfloat16):
            for name, err in example(dtype=dtype, seed=size["T"], **size).items():
                print(f"{size['T']} tokens, {dtype}: {name} {err:.4f} off the unquantized layer", flush=True)
