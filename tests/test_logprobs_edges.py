"""Token log probabilities at their edges: where tensors lie, magnitudes of logits, the ends of rows, ties, and the forms
over a head projection."""

import pytest
import torch

from optimus_dl_b200.ops.cross_entropy import linear_token_loss


# ------------------------------------------------------------------------------------------------ where tensors lie
def test_the_entropy_weight_has_to_be_where_the_rows_are():
    x, w = torch.randn(6, 16), torch.randn(9, 16)
    t, ew = torch.randint(0, 9, (6,)), torch.randn(6)
    zero = lambda n, a, b: (torch.zeros_like(n), torch.zeros_like(n))                          # noqa: E731
    linear_token_loss(x, w, t, zero, entropy_weight=ew)
    for bad in (dict(entropy_weight=ew.to("meta")), dict(entropy_weight=ew, t=t.to("meta")),
                dict(entropy_weight=ew, w=w.to("meta")), dict(entropy_weight=ew[:4], t=t[:4])):
        with pytest.raises(ValueError):
            linear_token_loss(x, bad.get("w", w), bad.get("t", t), zero, entropy_weight=bad["entropy_weight"])
