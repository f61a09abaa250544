"""Generation's C entry points as their header allows and the Python functions do not call them: results in the place of an
operand, workspaces kept by the caller, values near the ends of fp32's range."""
import pytest
import torch

from pragnosia_amd import fp4, rules
from pragnosia_amd._lib import check as ok, gen_lib
from pragnosia_amd.head import _raw_stream

from test_gpu_fp4 import BF16, F32, check, layer_norm, linear64, rows, weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,N", [(1, 40), (3, 77), (16, 2000), (32, 2321), (100, 2400), (330, 3016), (1001, 2203)])
def test_linear_into_its_residual(n, N, dtype):
    """y is resid, at every form of the kernels."""
    K = 264
    Q, x, ln, b, r = fp4.quantize(weight(N, K, dtype), 64), rows(n, K, dtype), layer_norm(K, dtype), rows(1, N, dtype, 3)[0], \
        rows(n, N, dtype, 4)
    for norm, act in ((None, 0), (ln, 1)):
        want = fp4.linear(x, Q, b, norm=norm, act="gelu" if act else None, resid=r)
        y = r.clone()
        lw, lb = (None, None) if norm is None else (norm.weight.data_ptr(), norm.bias.data_ptr())
        ok(gen_lib().pragnosia_fp4_linear(x.data_ptr(), dtype == BF16, Q.codes.data_ptr(), Q.scales.data_ptr(), lw, lb, 1e-5,
                                          b.data_ptr(), act, y.data_ptr(), y.data_ptr(), n, N, K, 64, _raw_stream(0)), "linear")
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V", [(1, 500), (5, 8193), (3, 40003), (16, 70001), (181, 40003)])
def test_rules_in_place(B, V, dtype):
    """out is the logits, with rows that start anywhere in a vector and share it with their neighbours."""
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = (3 * torch.randn(B, V, generator=g, device=DEV)).to(dtype)
    history = torch.randint(0, V, (B, 200), generator=g, device=DEV)
    mask = torch.randint(0, 1 << 32, (3, (V + 31) // 32), generator=g, device=DEV).to(torch.int32)
    state = torch.randint(-1, 4, (B,), generator=g, device=DEV)
    want = rules.apply_rules(logits, history, repetition=1.3, presence=0.5, frequency=0.25, mask=mask, state=state)
    ok(gen_lib().pragnosia_rules(logits.data_ptr(), dtype == BF16, history.data_ptr(), 200, 200, None, None, None, 1.3, None, 0.5,
                                 None, 0.25, None, None, 0, 0, mask.data_ptr(), 3, state.data_ptr(), logits.data_ptr(), None,
                                 None, 0, B, V, _raw_stream(0)), "rules")
    assert torch.equal(logits, want)


def test_a_workspace_of_other_calls():
    """What a workspace holds does not matter, nor who used it before."""
    g = torch.Generator(device=DEV).manual_seed(1)
    L = gen_lib()
    ws = torch.full((L.pragnosia_rules_workspace_bytes(9, 131072),), 255, dtype=torch.uint8, device=DEV)
    for B, V in ((9, 131072), (4, 40003), (9, 70001), (1, 131072)):
        x = torch.randn(B, V, generator=g, device=DEV)
        token = torch.empty(B, dtype=torch.long, device=DEV)
        ok(L.pragnosia_rules(x.data_ptr(), 0, None, 0, 0, None, None, None, 1.0, None, 0.0, None, 0.0, None, None, 0, 0, None, 0,
                             None, None, token.data_ptr(), ws.data_ptr(), ws.numel(), B, V, _raw_stream(0)), "rules")
        assert torch.equal(token, x.argmax(1))


@pytest.mark.parametrize("n,N", [(1, 40), (4, 40), (16, 40), (32, 2320), (100, 2400), (330, 3016), (1000, 2200)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("up", [-120, -95, 100])
def test_linear_far_from_one(n, N, up, dtype):
    """Rows of about 2^up and weights of about 2^-up: the products are ordinary numbers, and no part of a row is lost but what
    lies below 2^-126, the smallest normal bf16 number, in each of its three parts."""
    K = 264
    Q = fp4.quantize((weight(N, K, F32) * 2.0 ** min(-up, 110)).to(dtype), 64)
    x = (rows(n, K, F32) * 2.0 ** up).to(dtype)
    want, bound = linear64(x, Q)
    bound = bound + 3 * 2.0 ** -126 * fp4.dequantize(Q, F32).double().abs().sum(1)
    off = (fp4.linear(x, Q).double() - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} of the bound"
