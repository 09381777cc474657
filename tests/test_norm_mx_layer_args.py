"""What the norm, microscaled and routed-layer entry points refuse, before any device work, and what their size
queries say (no GPU needed)."""
import ctypes

import pytest

import tier_amd

F32, F16, BF16, Q8 = tier_amd.F32, tier_amd.F16, tier_amd.BF16, tier_amd.Q8_0
E2M1, E4M3 = tier_amd.MX_E2M1, tier_amd.MX_E4M3
EINVAL, UNSUPPORTED, OK = tier_amd.EINVAL, tier_amd.UNSUPPORTED, tier_amd.OK
A = 4096  # an address that no call follows


def L():
    return tier_amd.lib()


def norm(x=A, t=F32, ldx=300, r=A, ldr=300, g=A, eps=1e-5, h=A, ldh=300, y=A, ldy=300, q=A, rb=384, s=A, rs=A, M=2, K=300):
    return L().tiermm_rms_norm(x, t, ldx, r, ldr, g, eps, h, ldh, y, ldy, q, rb, s, rs, M, K, None)


def norm_mx(x=A, t=F32, ldx=300, r=A, ldr=300, g=A, eps=1e-5, h=A, ldh=300, y=A, ldy=300, f=E4M3, q=A, rb=512, s=A, sb=16,
            rs=A, M=2, K=300):
    return L().tiermm_rms_norm_mx(x, t, ldx, r, ldr, g, eps, h, ldh, y, ldy, f, q, rb, s, sb, rs, M, K, None)


def grad(dy=A, t=F32, ldy=300, h=A, ldh=300, g=A, rs=A, dh=A, lddh=300, dx=A, lddx=300, dg=A, M=2, K=300, ws=None, n=0):
    return L().tiermm_rms_norm_grad(dy, t, ldy, h, ldh, g, rs, dh, lddh, dx, lddx, dg, M, K, ws, n, None)


def mxq(x=A, t=F32, ldx=300, f=E2M1, q=A, rb=256, s=A, sb=16, M=2, K=300):
    return L().tiermm_mx_quant(x, t, ldx, f, q, rb, s, sb, M, K, None)


def blocks(w=A, rb=153, q=A, rbq=256, s=A, sb=16, N=2, K=288):
    return L().tiermm_mx_from_mxfp4(w, rb, q, rbq, s, sb, N, K, None)


def gemm(x=A, f=E2M1, rbx=256, sx=A, sbx=16, w=A, rbw=256, sw=A, sbw=16, b=None, y=A, t=F32, ldy=20, M=2, N=20, K=300):
    return L().tiermm_mx_gemm(x, f, rbx, sx, sbx, w, rbw, sw, sbw, b, y, t, ldy, M, N, K, None)


def linear(x=A, xt=F32, ldx=300, f=E4M3, w=A, rbw=256, sw=A, sbw=16, b=None, y=A, t=F32, ldy=20, M=2, N=20, K=300, ws=None, n=0):
    return L().tiermm_mx_linear(x, xt, ldx, f, w, rbw, sw, sbw, b, y, t, ldy, M, N, K, ws, n, None)


def layer(x=A, rbx=384, sx=A, ids=A, w=A, g=A, rbg=384, sg=A, d=A, rbd=128, sd=A, o=A, t=F32, ldo=300, T=2, k=2, E=4, K=300,
          F=100, ws=None, n=0):
    return L().tiermm_moe_i8_layer(x, rbx, sx, ids, w, g, rbg, sg, d, rbd, sd, o, t, ldo, T, k, E, K, F, ws, n, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call", [norm, norm_mx])
@pytest.mark.parametrize("kw,code", [
    ({"t": Q8}, UNSUPPORTED), ({"M": -1}, EINVAL), ({"K": 0}, EINVAL), ({"K": -5}, EINVAL), ({"M": (1 << 23) + 1}, UNSUPPORTED),
    ({"K": (1 << 20) + 1, "ldx": 1 << 21, "ldr": 1 << 21, "ldh": 1 << 21, "ldy": 1 << 21}, UNSUPPORTED),
    ({"eps": -1e-9}, EINVAL), ({"eps": NAN}, EINVAL), ({"eps": INF}, EINVAL),
    ({"ldx": 299}, EINVAL), ({"ldr": 299}, EINVAL), ({"ldh": 299}, EINVAL), ({"ldy": 299}, EINVAL), ({"ldx": -16}, EINVAL),
    ({"x": None}, EINVAL), ({"g": None}, EINVAL), ({"x": A + 2}, EINVAL), ({"r": A + 1}, EINVAL), ({"g": A + 2}, EINVAL),
    ({"h": A + 1, "t": F16}, EINVAL), ({"y": A + 3}, EINVAL), ({"rs": A + 2}, EINVAL), ({"s": None}, EINVAL),
    ({"q": A + 8}, EINVAL), ({"rb": 256}, EINVAL), ({"rb": 520}, EINVAL), ({"rb": 1 << 62}, EINVAL)])
def test_norms_refuse(call, kw, code):
    assert call(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [({"s": A + 2}, EINVAL), ({"K": 133121, "ldx": 1 << 18, "ldr": 1 << 18, "ldh": 1 << 18,
                                                               "ldy": 1 << 18, "rb": 1 << 18}, UNSUPPORTED)])
def test_int8_norm_refuses(kw, code):
    assert norm(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [({"f": 6}, UNSUPPORTED), ({"f": 0}, UNSUPPORTED), ({"q": None}, EINVAL), ({"s": A + 8}, EINVAL),
                                     ({"sb": 8}, EINVAL), ({"sb": 24}, EINVAL), ({"sb": -16}, EINVAL)])
def test_mx_norm_refuses(kw, code):
    assert norm_mx(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"t": 99}, UNSUPPORTED), ({"M": -1}, EINVAL), ({"K": 0}, EINVAL), ({"M": (1 << 23) + 1}, UNSUPPORTED), ({"ldy": 299}, EINVAL),
    ({"ldh": 1}, EINVAL), ({"lddh": 299}, EINVAL), ({"lddx": 0}, EINVAL), ({"lddx": 1 << 62}, EINVAL), ({"dy": None}, EINVAL),
    ({"h": None}, EINVAL), ({"g": None}, EINVAL), ({"rs": None}, EINVAL), ({"dx": None}, EINVAL), ({"dy": A + 2}, EINVAL),
    ({"h": A + 1}, EINVAL), ({"dh": A + 1, "t": BF16}, EINVAL), ({"dx": A + 2}, EINVAL), ({"g": A + 1}, EINVAL),
    ({"rs": A + 2}, EINVAL), ({"dg": A + 2}, EINVAL), ({"ws": A, "n": 16}, EINVAL), ({"ws": A + 2, "n": 1 << 20}, EINVAL)])
def test_gradient_refuses(kw, code):
    assert grad(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"t": Q8}, UNSUPPORTED), ({"f": 5}, UNSUPPORTED), ({"M": -1}, EINVAL), ({"K": 0}, EINVAL),
    ({"K": (1 << 20) + 1, "ldx": 1 << 21}, UNSUPPORTED), ({"M": (1 << 20) + 1}, UNSUPPORTED), ({"ldx": 299}, EINVAL),
    ({"ldx": -1}, EINVAL), ({"x": None}, EINVAL), ({"x": A + 1, "t": F16}, EINVAL), ({"q": None}, EINVAL), ({"s": None}, EINVAL),
    ({"q": A + 4}, EINVAL), ({"s": A + 1}, EINVAL), ({"rb": 240}, EINVAL), ({"rb": 264}, EINVAL), ({"sb": 0}, EINVAL),
    ({"sb": 17}, EINVAL), ({"f": E4M3}, EINVAL)])
def test_mx_quant_refuses(kw, code):
    assert mxq(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"N": -1}, EINVAL), ({"K": 0}, EINVAL), ({"K": 300}, UNSUPPORTED), ({"rb": 152}, EINVAL), ({"rb": -17}, EINVAL),
    ({"w": None}, EINVAL), ({"q": None}, EINVAL), ({"s": None}, EINVAL), ({"rbq": 128}, EINVAL), ({"sb": 8}, EINVAL),
    ({"q": A + 8}, EINVAL)])
def test_from_mxfp4_refuses(kw, code):
    assert blocks(**kw) == code and tier_amd.last_error()


SIDE = [({"f": 3}, UNSUPPORTED), ({"M": -1}, EINVAL), ({"N": -1}, EINVAL), ({"K": 0}, EINVAL), ({"M": (1 << 20) + 1}, UNSUPPORTED),
        ({"N": (1 << 26) + 1}, UNSUPPORTED), ({"K": (1 << 20) + 1, "ldx": 1 << 21}, UNSUPPORTED), ({"t": Q8}, UNSUPPORTED),
        ({"ldy": 19}, EINVAL), ({"ldy": -20}, EINVAL), ({"y": None}, EINVAL), ({"y": A + 2}, EINVAL), ({"x": None}, EINVAL),
        ({"w": None}, EINVAL), ({"sw": None}, EINVAL), ({"w": A + 8}, EINVAL), ({"sw": A + 4}, EINVAL), ({"rbw": 240}, EINVAL),
        ({"rbw": 257}, EINVAL), ({"sbw": 8}, EINVAL), ({"sbw": 1 << 62}, EINVAL), ({"b": A + 2}, EINVAL)]


@pytest.mark.parametrize("call", [gemm, linear])
@pytest.mark.parametrize("kw,code", SIDE)
def test_mx_products_refuse(call, kw, code):
    if call is gemm:
        kw = {k: v for k, v in kw.items() if k != "ldx"}
    assert call(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("call,kw,code", [
    (gemm, {"x": A + 8}, EINVAL), (gemm, {"sx": None}, EINVAL), (gemm, {"sx": A + 2}, EINVAL), (gemm, {"rbx": 248}, EINVAL),
    (gemm, {"sbx": 15}, EINVAL), (gemm, {"f": E4M3}, EINVAL), (linear, {"xt": Q8}, UNSUPPORTED), (linear, {"ldx": 299}, EINVAL),
    (linear, {"x": A + 2}, EINVAL), (linear, {"ws": A + 8, "n": 1 << 20}, EINVAL),
    (linear, {"M": 40, "ws": A, "n": 40 * (512 + 16) - 1}, EINVAL)])
def test_mx_products_refuse_their_own(call, kw, code):
    assert call(**kw) == code and tier_amd.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"T": -1}, EINVAL), ({"k": -1}, EINVAL), ({"E": 0}, EINVAL), ({"K": 0}, EINVAL), ({"F": -1}, EINVAL), ({"T": 65}, UNSUPPORTED),
    ({"k": 33}, UNSUPPORTED), ({"E": 1025}, UNSUPPORTED), ({"K": 133121, "rbx": 1 << 18, "rbg": 1 << 18, "ldo": 1 << 18}, UNSUPPORTED),
    ({"F": 133121, "rbd": 1 << 18}, UNSUPPORTED), ({"t": Q8}, UNSUPPORTED), ({"ldo": 299}, EINVAL), ({"ldo": -300}, EINVAL),
    ({"o": None}, EINVAL), ({"o": A + 2}, EINVAL), ({"x": None}, EINVAL), ({"g": None}, EINVAL), ({"d": None}, EINVAL),
    ({"x": A + 4}, EINVAL), ({"g": A + 8}, EINVAL), ({"d": A + 1}, EINVAL), ({"rbx": 368}, EINVAL), ({"rbg": 300}, EINVAL),
    ({"rbg": 392}, EINVAL), ({"rbd": 112}, EINVAL), ({"rbd": 1 << 62}, EINVAL), ({"sx": None}, EINVAL), ({"ids": None}, EINVAL),
    ({"w": None}, EINVAL), ({"sg": None}, EINVAL), ({"sd": None}, EINVAL), ({"sx": A + 2}, EINVAL), ({"ids": A + 1}, EINVAL),
    ({"w": A + 2}, EINVAL), ({"sg": A + 3}, EINVAL), ({"sd": A + 2}, EINVAL), ({"ws": A + 8, "n": 1 << 20}, EINVAL),
    ({"ws": A, "n": 64}, EINVAL)])
def test_layer_refuses(kw, code):
    assert layer(**kw) == code and tier_amd.last_error()


def test_empty_calls():
    assert norm(M=0, x=None, g=None, h=None, y=None, q=None) == norm_mx(M=0, x=None, q=None, s=None) == OK
    assert grad(M=0, dg=None, dy=None) == mxq(M=0, x=None, q=None) == blocks(N=0, w=None) == OK
    assert gemm(M=0, x=None) == gemm(N=0, w=None, ldy=0) == linear(M=0, x=None) == linear(N=0, y=None, ldy=0) == OK
    assert layer(T=0, x=None, o=None) == OK


def test_sizes():
    assert tier_amd.mx_row_bytes(E2M1, 5120) == 2560 and tier_amd.mx_row_bytes(E4M3, 5120) == 5120
    assert tier_amd.mx_row_bytes(E2M1, 1) == 128 and tier_amd.mx_row_bytes(E4M3, 257) == 512
    assert tier_amd.mx_row_bytes(5, 256) == tier_amd.mx_row_bytes(E2M1, 0) == tier_amd.mx_row_bytes(E2M1, (1 << 20) + 1) == 0
    assert tier_amd.mx_scale_bytes(5120) == 160 and tier_amd.mx_scale_bytes(1) == 16 and tier_amd.mx_scale_bytes(513) == 32
    assert tier_amd.mx_scale_bytes(0) == tier_amd.mx_scale_bytes((1 << 20) + 1) == 0
    assert tier_amd.mx_linear_ws_bytes(E4M3, 40, 20, 300) >= 40 * (512 + 16) and tier_amd.mx_linear_ws_bytes(3, 4, 4, 4) == 0
    assert tier_amd.mx_linear_ws_bytes(E4M3, 0, 20, 300) == tier_amd.mx_linear_ws_bytes(E4M3, 4, 20, 0) == 0
    assert tier_amd.rms_norm_grad_ws_bytes(4, 300) >= 4 * 300 * 4 and tier_amd.rms_norm_grad_ws_bytes(0, 300) == 0
    assert tier_amd.moe_i8_layer_ws_bytes(1, 8, 2048, 1408) > 0
    assert tier_amd.moe_i8_layer_ws_bytes(65, 8, 2048, 1408) == tier_amd.moe_i8_layer_ws_bytes(4, 8, 0, 8) == 0


# wrapper -> arguments that it refuses or answers before any device work
CALLS = {
    "rms_norm": (A, F32, 300, None, 0, A, 1e-5, None, 0, None, 0, None, 0, None, None, 0, 300),
    "rms_norm_mx": (A, F32, 300, None, 0, A, 1e-5, None, 0, None, 0, E4M3, A, 512, A, 16, None, 0, 300),
    "rms_norm_grad": (A, F32, 300, A, 300, A, A, None, 0, A, 300, None, 0, 300, None, 0),
    "mx_quant": (A, F32, 300, E2M1, A, 256, A, 16, 0, 300),
    "mx_from_mxfp4": (A, 153, A, 256, A, 16, 0, 288),
    "mx_gemm": (A, E2M1, 256, A, 16, A, 256, A, 16, None, A, F32, 20, 0, 20, 300),
    "mx_linear": (A, F32, 300, E2M1, A, 256, A, 16, None, A, F32, 20, 0, 20, 300, None, 0),
    "moe_i8_layer": (A, 384, A, A, A, A, 384, A, A, 128, A, A, F32, 300, 0, 2, 4, 300, 100, None, 0),
}


@pytest.mark.parametrize("name", CALLS)
def test_none_is_no_number(name):
    """None is a null address and not a size, a stride, a type or eps; a float is no size."""
    args, types = CALLS[name], getattr(tier_amd.lib(), "tiermm_" + name).argtypes
    assert len(types) == len(args) + 1  # the stream
    getattr(tier_amd, name)(*args)
    for i, t in enumerate(types[:-1]):
        with_none = args[:i] + (None,) + args[i + 1:]
        if t is ctypes.c_void_p:
            getattr(tier_amd, name)(*with_none)
        else:
            with pytest.raises((TypeError, ctypes.ArgumentError)):
                getattr(tier_amd, name)(*with_none)
            if t is not ctypes.c_float:
                with pytest.raises((TypeError, ctypes.ArgumentError)):
                    getattr(tier_amd, name)(*(args[:i] + (1.5,) + args[i + 1:]))


def test_float_arguments_arrive():
    """eps through both ways of calling: its sign and its NaN are seen."""
    for eps in (-1.0, float("nan"), float("inf")):
        a = list(CALLS["rms_norm"])
        a[6] = eps
        with pytest.raises(tier_amd.TiermmError) as e:
            tier_amd.rms_norm(*a)
        assert e.value.code == EINVAL and "eps" in str(e.value)
    a[6] = 1  # whole numbers are floats too
    tier_amd.rms_norm(*a)


@pytest.mark.parametrize("call,name", [(norm, "ldx"), (norm, "ldr"), (norm, "ldh"), (norm, "ldy"), (norm, "rb"), (norm_mx, "rb"),
                                       (norm_mx, "sb"), (grad, "ldy"), (grad, "ldh"), (grad, "lddh"), (grad, "lddx"), (mxq, "ldx"),
                                       (mxq, "rb"), (mxq, "sb"), (blocks, "rb"), (blocks, "rbq"), (blocks, "sb"), (gemm, "rbx"),
                                       (gemm, "sbx"), (gemm, "rbw"), (gemm, "sbw"), (gemm, "ldy"), (linear, "ldx"), (linear, "rbw"),
                                       (linear, "sbw"), (linear, "ldy"), (layer, "rbx"), (layer, "rbg"), (layer, "rbd"),
                                       (layer, "ldo")], ids=lambda v: getattr(v, "__name__", v))
@pytest.mark.parametrize("stride", [-16, -(1 << 62), 1 << 62, (1 << 40) + 16])
def test_strides_past_any_memory(call, name, stride):
    assert call(**{name: stride}) == EINVAL and tier_amd.last_error()


# A launch has less than 2^32 threads: 1024 for a row of a norm, 256 for a row of blocks.
@pytest.mark.parametrize("call,kw", [(norm, {"M": 1 << 22}), (norm_mx, {"M": 1 << 22}), (grad, {"M": 1 << 22}),
                                     (blocks, {"N": 1 << 24}), (gemm, {"N": 1 << 24, "ldy": 1 << 24}),
                                     (linear, {"N": 1 << 24, "ldy": 1 << 24})])
def test_more_rows_than_a_launch_has_threads_for(call, kw):
    assert call(**kw) == UNSUPPORTED and "at most" in tier_amd.last_error()
    assert tier_amd.rms_norm_grad_ws_bytes(1 << 22, 300) == 0
