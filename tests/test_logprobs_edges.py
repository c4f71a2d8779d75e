"""Token log probabilities at their edges: where tensors lie, magnitudes of logits, the ends of rows, ties, and the forms
over a head projection."""

import pytest
import torch

from optimus_dl_b200.ops import logprobs as lp
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


def test_the_head_has_to_fit_the_rows_and_be_where_they_are():
    x, w, t = torch.randn(6, 16), torch.randn(9, 16), torch.randint(0, 9, (6,))
    for bad in (w.to("meta"), w[:, :8], w[0], w[None]):
        with pytest.raises(ValueError):
            lp.linear_token_logprobs(x, bad, t)


def test_the_head_projection_runs_on_the_rows_own_device(monkeypatch):
    """Of the two launches the product alone would go to the current device. Tensors without memory stand for those of a
    second GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    entered, inside = [], []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *exc):
            entered.pop()

    def product(a, b, out):
        inside.append(list(entered))

    def scores(z, t, **kw):
        n = z.new_empty(t.shape, dtype=torch.float32)
        return lp.TokenLogprobs(n, n, None, None)

    monkeypatch.setattr(lp._lib, "on_device", On)
    monkeypatch.setattr(lp.gemm, "gemm", product)
    monkeypatch.setattr(lp, "token_logprobs", scores)
    with FakeTensorMode():
        there = torch.device("cuda", 1)
        x, w = (torch.empty(n, 16, dtype=torch.bfloat16, device=there) for n in (6, 9))
        r = lp.linear_token_logprobs(x, w, torch.zeros(6, dtype=torch.int64, device=there), chunk_rows=4)
    assert r.logp.shape == (6,) and inside == [[there], [there]]


# ------------------------------------------------------------------------------------------------ ends of rows, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,temperature", [(30.0, 1e-6), (7e5, 1.0), (60000.0, 0.1), (50.0, 7e-5)])
def test_a_maximum_at_either_end_of_a_row(dtype, size, temperature):
    """Alone with the distribution: its entropy is 0 wherever it stands, to what the logarithm and the reference's own
    rounding leave, 2^-20 of the exponent's residue (at most 2) and of 1."""
    if size > torch.finfo(dtype).max:
        pytest.skip("not a number of this type")
    for vocab in (1025, 1027, 4099, 20003):
        z = torch.zeros(24, vocab)
        for i in range(24):
            z[i, [0, 1, 2, 3, 6, 7, vocab // 2, vocab - 8, vocab - 7, vocab - 3, vocab - 2, vocab - 1][i % 12]] = size + i
        r = lp.token_logprobs(z.to(dtype).cuda(), z.argmax(-1).cuda(), temperature=temperature)
        assert float(r.entropy.abs().max()) <= 5e-5 and float(r.logp.abs().max()) <= 5e-5
