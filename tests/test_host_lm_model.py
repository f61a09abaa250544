"""CPU checks of the LM class around its two ends."""
import io

import torch

from pragnosia_amd.model import LM


def test_model_saved_before_the_switch():
    """An LM saved whole by a version without fused_ends loads and gives its loss as it did."""
    torch.manual_seed(0)
    m = LM(vocab=40, d=64, layers=1, ctx=16)
    h, y = torch.randn(2, 16, 64), torch.randint(0, 40, (2, 16))
    want = m.loss(h, y)
    old = {k: v for k, v in m.__dict__.items() if k != "fused_ends"}
    m.__dict__.clear()
    m.__dict__.update(old)
    for e in (m.e, m.p):
        e.__dict__.pop("sorted_grad", None)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    back = torch.load(f, weights_only=False)
    assert "fused_ends" not in back.__dict__ and torch.equal(back.loss(h, y), want)
    assert torch.equal(back.e(y), m.e(y))
