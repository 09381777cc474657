"""Row strides that are negative numbers taken for sizes (or as large): refused on the host, in front of
any device work, by every routed-row and int8 entry point (no GPU needed)."""
import pytest

import tier_amd
from test_routed_i8_args import gemm, grouped, linear, quant, sort, sort_grad, unsort, unsort_grad

EINVAL = tier_amd.EINVAL
STRIDES = [(sort, "ldx"), (sort, "lds"), (sort_grad, "ldx"), (sort_grad, "lds"), (unsort, "lds"), (unsort, "ldo"),
           (unsort_grad, "ldo"), (unsort_grad, "lds"), (unsort_grad, "ldd"), (quant, "ldx"), (quant, "rb"), (gemm, "rbx"),
           (gemm, "rbw"), (gemm, "ldy"), (linear, "ldx"), (linear, "rbw"), (linear, "ldy"), (grouped, "rbx"),
           (grouped, "rbw"), (grouped, "ldy")]


@pytest.mark.parametrize("call,name", STRIDES, ids=lambda v: getattr(v, "__name__", v))
@pytest.mark.parametrize("stride", [-16, -(1 << 62), 1 << 62, (1 << 40) + 16])
def test_strides_past_any_memory(call, name, stride):
    assert call(**{name: stride}) == EINVAL and tier_amd.last_error()
