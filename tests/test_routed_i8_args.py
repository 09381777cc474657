"""What the routed-row and int8 entry points refuse, before any device work (no GPU needed)."""
import pytest

import tier_amd

F32, F16, BF16, Q8 = tier_amd.F32, tier_amd.F16, tier_amd.BF16, tier_amd.Q8_0
EINVAL, UNSUPPORTED, OK = tier_amd.EINVAL, tier_amd.UNSUPPORTED, tier_amd.OK
A = 4096  # an address that no call follows


def L():
    return tier_amd.lib()


def plan(ids=A, T=4, k=2, E=8, off=A, tp=A, sp=A, ws=None, n=0):
    return L().tiermm_moe_plan(ids, T, k, E, off, tp, sp, ws, n, None)


@pytest.mark.parametrize("kw,code", [
    ({"T": -1}, EINVAL), ({"k": -1}, EINVAL), ({"E": 0}, EINVAL), ({"E": 1025}, UNSUPPORTED),
    ({"T": 1 << 21, "k": 8}, UNSUPPORTED), ({"T": 0x7fffffff, "k": 0x7fffffff}, UNSUPPORTED),
    ({"ids": None}, EINVAL), ({"off": None}, EINVAL), ({"tp": None}, EINVAL), ({"sp": None}, EINVAL),
    ({"ids": A + 2}, EINVAL), ({"off": A + 1}, EINVAL), ({"tp": A + 3}, EINVAL), ({"sp": A + 2}, EINVAL),
    ({"T": 20000, "k": 8, "ws": A, "n": 16}, EINVAL)])
def test_plan_refuses(kw, code):
    assert plan(**kw) == code and tier_amd.last_error()


def test_plan_workspace():
    assert tier_amd.moe_plan_ws_bytes(4096, 8, 64) == 0
    assert tier_amd.moe_plan_ws_bytes(4097, 8, 64) > 0
    assert tier_amd.moe_plan_ws_bytes(-1, 8, 64) == 0


def sort(x=A, t=F32, ldx=16, tp=A, sp=A, y=A, lds=16, T=4, k=2, K=16):
    return L().tiermm_moe_sort(x, t, ldx, tp, sp, y, lds, T, k, K, None)


def sort_grad(x=A, t=F32, lds=16, tp=A, y=A, ldx=16, T=4, k=2, K=16):
    return L().tiermm_moe_sort_grad(x, t, lds, tp, y, ldx, T, k, K, None)


def unsort(x=A, t=F32, lds=16, tp=A, w=A, y=A, ldo=16, T=4, k=2, K=16):
    return L().tiermm_moe_unsort(x, t, lds, tp, w, y, ldo, T, k, K, None)


def unsort_grad(d=A, t=F32, ldo=16, x=A, lds=16, tp=A, sp=A, w=A, y=A, ldd=16, dw=A, T=4, k=2, K=16):
    return L().tiermm_moe_unsort_grad(d, t, ldo, x, lds, tp, sp, w, y, ldd, dw, T, k, K, None)


@pytest.mark.parametrize("call", [sort, sort_grad, unsort, unsort_grad])
@pytest.mark.parametrize("kw,code", [
    ({"t": Q8}, UNSUPPORTED), ({"t": 99}, UNSUPPORTED), ({"T": -1}, EINVAL), ({"k": -2}, EINVAL), ({"K": -1}, EINVAL),
    ({"lds": 15}, EINVAL), ({"T": 1 << 22, "k": 8}, UNSUPPORTED), ({"T": (1 << 23) + 1, "k": 0}, UNSUPPORTED),
    ({"x": None}, EINVAL), ({"y": None}, EINVAL), ({"tp": None}, EINVAL), ({"x": A + 2}, EINVAL),
    ({"y": A + 1, "t": F16}, EINVAL), ({"tp": A + 2}, EINVAL)])
def test_rows_refuse(call, kw, code):
    assert call(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("call,kw", [(sort, {"ldx": 15}), (sort, {"sp": None}), (sort, {"sp": A + 1}),
                                     (sort_grad, {"ldx": 15}), (unsort, {"ldo": 3}), (unsort, {"w": None}),
                                     (unsort, {"w": A + 2}), (unsort_grad, {"ldo": 1}), (unsort_grad, {"ldd": 15}),
                                     (unsort_grad, {"d": None}), (unsort_grad, {"dw": None}),
                                     (unsort_grad, {"dw": A + 2}), (unsort_grad, {"sp": None}),
                                     (unsort_grad, {"w": None}), (unsort_grad, {"d": A + 1, "t": BF16})])
def test_rows_refuse_their_own(call, kw):
    assert call(**kw) == EINVAL and tier_amd.last_error()


def test_empty_row_calls():
    assert sort(T=0, x=None, y=None, tp=None, sp=None) == OK
    assert sort(k=0) == sort(K=0) == OK
    assert sort_grad(T=0) == sort_grad(K=0) == unsort(T=0) == unsort(K=0) == OK
    assert unsort_grad(T=0) == unsort_grad(k=0) == OK


def quant(x=A, t=F32, ldx=300, q=A, rb=384, s=A, M=2, K=300):
    return L().tiermm_i8_quant(x, t, ldx, q, rb, s, M, K, None)


def gemm(x=A, rbx=384, sx=A, w=A, rbw=384, sw=A, b=None, y=A, t=F32, ldy=20, M=2, N=20, K=300):
    return L().tiermm_i8_gemm(x, rbx, sx, w, rbw, sw, b, y, t, ldy, M, N, K, None)


def linear(x=A, xt=F32, ldx=300, w=A, rbw=384, sw=A, b=None, y=A, t=F32, ldy=20, M=2, N=20, K=300, ws=A, n=1 << 20):
    return L().tiermm_i8_linear(x, xt, ldx, w, rbw, sw, b, y, t, ldy, M, N, K, ws, n, None)


def grouped(x=A, rbx=384, sx=A, rows=A, T=2, k=2, off=A, E=4, w=A, rbw=384, sw=A, y=A, t=F32, ldy=20, M=4, N=20, K=300):
    return L().tiermm_i8_gemm_grouped(x, rbx, sx, rows, T, k, off, E, w, rbw, sw, y, t, ldy, M, N, K, None)


@pytest.mark.parametrize("kw,code", [
    ({"M": -1}, EINVAL), ({"K": 0}, EINVAL), ({"K": 133121, "ldx": 133121, "rb": 133248}, UNSUPPORTED),
    ({"M": (1 << 23) + 1}, UNSUPPORTED), ({"t": Q8}, UNSUPPORTED), ({"ldx": 299}, EINVAL), ({"rb": 300}, EINVAL),
    ({"rb": 385}, EINVAL), ({"q": A + 8}, EINVAL), ({"q": None}, EINVAL), ({"x": None}, EINVAL), ({"x": A + 2}, EINVAL),
    ({"s": None}, EINVAL), ({"s": A + 2}, EINVAL)])
def test_quant_refuses(kw, code):
    assert quant(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("call", [gemm, linear, grouped])
@pytest.mark.parametrize("kw,code", [
    ({"M": -1}, EINVAL), ({"N": -1}, EINVAL), ({"K": -3}, EINVAL), ({"K": 140000}, UNSUPPORTED), ({"t": Q8}, UNSUPPORTED),
    ({"ldy": 19}, EINVAL), ({"y": None}, EINVAL), ({"y": A + 1, "t": F16}, EINVAL), ({"rbw": 256}, EINVAL),
    ({"N": (1 << 26) + 1, "ldy": 1 << 27}, UNSUPPORTED), ({"M": (1 << 23) + 1}, UNSUPPORTED),
    ({"rbw": 390}, EINVAL), ({"w": A + 4}, EINVAL), ({"w": None}, EINVAL), ({"sw": None}, EINVAL),
    ({"sw": A + 1}, EINVAL), ({"x": None}, EINVAL)])
def test_products_refuse(call, kw, code):
    assert call(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("call,kw,code", [
    (gemm, {"rbx": 300}, EINVAL), (gemm, {"x": A + 8}, EINVAL), (gemm, {"sx": None}, EINVAL), (gemm, {"b": A + 2}, EINVAL),
    (linear, {"xt": 99}, UNSUPPORTED), (linear, {"ldx": 299}, EINVAL), (linear, {"x": A + 2}, EINVAL),
    (linear, {"ws": A + 4}, EINVAL), (linear, {"b": A + 1}, EINVAL), (linear, {"M": 200, "n": 64}, EINVAL),
    (grouped, {"rbx": 128}, EINVAL), (grouped, {"T": -1}, EINVAL), (grouped, {"T": 0}, EINVAL), (grouped, {"k": 0}, EINVAL),
    (grouped, {"E": 0}, EINVAL), (grouped, {"E": 2000}, UNSUPPORTED), (grouped, {"off": None}, EINVAL),
    (grouped, {"off": A + 2}, EINVAL), (grouped, {"rows": A + 1}, EINVAL), (grouped, {"sx": None}, EINVAL)])
def test_products_refuse_their_own(call, kw, code):
    assert call(**kw) == code and tier_amd.last_error()


def test_empty_products():
    assert quant(M=0, x=None) == gemm(M=0) == gemm(N=0) == linear(M=0) == linear(N=0) == OK
    assert grouped(M=0) == grouped(N=0) == OK


def test_row_bytes():
    assert [tier_amd.i8_row_bytes(K) for K in (1, 127, 128, 129, 5120, 1408, 133120, 133121, 0, -1)] == [
        128, 128, 128, 256, 5120, 1408, 133120, 0, 0, 0]
    assert tier_amd.i8_linear_ws_bytes(3, 5, 300) >= 3 * 384 + 12
    assert tier_amd.i8_linear_ws_bytes(0, 5, 300) == 0


def test_call_arguments():
    """tier_amd._call: integers of either sign, None as a null pointer, and nothing else."""
    from tier_amd import _call
    import ctypes
    f = _call.Call(ctypes.cast(L().tiermm_moe_plan, ctypes.c_void_p).value, 10)
    assert f(A, -1, 2, 8, A, A, A, None, 0, None) == EINVAL
    assert f(None, 4, 2, 8, A, A, A, None, 0, None) == EINVAL
    for bad in ((A,) * 9, (A,) * 11, ("x",) + (1,) * 9, (1.5,) + (1,) * 9):
        with pytest.raises(TypeError):
            f(*bad)
    with pytest.raises(TypeError):
        f(*(A,) * 9, stream=None)
    for address, n in ((0, 3), (16, -1), (16, 21)):
        with pytest.raises(ValueError):
            _call.Call(address, n)
    with pytest.raises(tier_amd.TiermmError):
        tier_amd.moe_plan(A, -1, 2, 8, A, A, A)
