"""Generation's operators at the largest sizes that they take."""
import math

import pytest
import torch

from pragnosia_amd import fp4, rules

from test_gpu_fp4 import BF16, F32, check, layer_norm, rows, weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,N", [(1, 40), (4, 40), (16, 40), (32, 2321), (100, 2407)])
def test_longest_rows(n, N, dtype):
    """65536 columns, the last block of which may be the only one a wave takes."""
    for K in (65536, 65408 + 8):
        Q = fp4.quantize(weight(N, K, dtype), 64)
        check(rows(n, K, dtype), Q)
        check(rows(n, K, dtype), Q, norm=layer_norm(K, dtype), act="gelu")


@pytest.mark.parametrize("n", [1, 4, 9])
def test_most_columns(n):
    """2^26 outputs: every row of the weight is told by its sign and size."""
    N, K = 1 << 26, 8
    sign = (torch.arange(N, device=DEV) % 7 < 3).float() * 2 - 1
    W = torch.zeros(N, K, device=DEV)
    W[:, 0], W[:, 5] = 6.0 * sign, 3.0
    Q = fp4.quantize(W, 128)
    assert torch.equal(fp4.dequantize(Q), W)
    del W
    x = torch.zeros(n, K, device=DEV)
    x[:, 0], x[:, 5] = torch.arange(1, n + 1, device=DEV), 2.0
    y = fp4.linear(x, Q)
    for i in range(n):
        assert torch.equal(y[i], 6.0 * (i + 1) * sign + 6.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_most_rows(dtype):
    """2^24 rows, each of whose results is one of its values."""
    n, N, K = 1 << 24, 16, 32
    W = torch.zeros(N, K, device=DEV, dtype=dtype)
    W[torch.arange(N, device=DEV), torch.arange(N, device=DEV) * 2 + 1] = 6.0
    Q = fp4.quantize(W, 32)
    x = torch.arange(n, device=DEV, dtype=torch.int32)[:, None].remainder(251).to(dtype) + torch.arange(K, device=DEV).to(dtype)
    y = fp4.linear(x, Q)
    for a in range(0, n, 1 << 21):
        assert torch.equal(y[a:a + (1 << 21)], (6.0 * x[a:a + (1 << 21), 1::2].float()).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_largest_vocabulary(dtype):
    B, V = 3, 1 << 26
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.zeros(B, V, device=DEV, dtype=dtype)
    x[0, V - 1], x[1, V - 1], x[1, 12345], x[2, V - 2] = 4.0, 4.0, 3.0, 2.0
    h = torch.randint(1 << 20, V - 2, (B, 500), generator=g, device=DEV)
    h[1, 7] = V - 1
    mask = torch.full((2, V // 32), -1, dtype=torch.int32, device=DEV)
    mask[1, -1] = 0x7fffffff >> 1  # (not the last two words)
    state = torch.tensor([0, 0, 1], device=DEV)
    kw = dict(repetition=2.0, presence=0.5, mask=mask, state=state)
    assert rules.next_token(x, h, **kw).tolist() == [V - 1, 12345, 0]
    out = rules.apply_rules(x, h, **kw)
    assert out[0, V - 1] == 4 and out[1, V - 1] == 1.5 and out[1, 12345] == 3
    assert (out[2, V - 2:] == -math.inf).all() and (out[2, :V - 2] > -math.inf).all()
    for b in range(B):  # (0 / 2 - 0.5, and once less the 0.5 for each further time: frequency is 0)
        assert (out[b, h[b]].float() <= 1.5).all() and (out[b] == -0.5).sum() == h[b][h[b] < V - 2].unique().numel()


def test_most_sequences():
    B, V = 65535, 40
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(B, V, generator=g, device=DEV)
    h = torch.randint(0, V, (B, 3), generator=g, device=DEV)
    got = rules.apply_rules(x, h, repetition=2.0)
    seen = torch.zeros(B, V, dtype=torch.bool, device=DEV).scatter_(1, h, True)
    want = torch.where(seen, torch.where(x > 0, x / 2, x * 2), x)
    assert torch.equal(got, want) and torch.equal(rules.next_token(x, h, repetition=2.0), want.argmax(1))
    long = torch.randn(65535, 33000, generator=g, device=DEV, dtype=F32).to(BF16)
    assert torch.equal(rules.next_token(long, h, repetition=1.0), long.float().argmax(1))


def test_longest_history():
    """2^24 tokens, some words most of them, under a list of as many entries as then fit."""
    L, V = 1 << 24, 9000
    h = torch.arange(L, device=DEV)[None] % 4096 % 3 + torch.arange(L, device=DEV)[None] // 4096 % 2 * 8990
    times = torch.bincount(h[0], minlength=V)
    assert times.sum() == L
    x = torch.zeros(1, V, device=DEV)
    ids = torch.arange(63, device=DEV) * 2
    kw = dict(presence=1.0, frequency=2.0 ** -10, bias=(ids, torch.arange(63.0, device=DEV)))
    want = -(times > 0).double() - times.double() * 2.0 ** -10
    want[ids] += torch.arange(63.0, device=DEV).double()
    got = rules.apply_rules(x, h, **kw)[0].double()
    assert ((got - want).abs() <= 3 * 2.0 ** -24 * (times * 2.0 ** -10 + 64)).all()
    assert rules.next_token(x, h, **kw).item() == 124
    with pytest.raises(rules.PragnosiaError, match="31 bits"):
        rules.apply_rules(x, h, bias=(torch.arange(64, device=DEV), torch.zeros(64, device=DEV)))
