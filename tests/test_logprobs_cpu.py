"""Log probabilities of given tokens on host tensors, and the refusals."""

import pytest
import torch

from zookeeper_amd.ops import token_logprobs


def test_values_and_alternatives():
    x = torch.tensor([[1.0, 3.0, 3.0, -1.0], [0.0, 0.0, 0.0, 0.0]], dtype=torch.float64)
    t = torch.tensor([1, 3])
    r = token_logprobs(x, t, top=3)
    lp = torch.log_softmax(x, -1)
    torch.testing.assert_close(r.logp, lp[[0, 1], [1, 3]])
    torch.testing.assert_close(r.entropy, -(lp.exp() * lp).sum(-1))
    assert r.top_ids.tolist() == [[1, 2, 0], [0, 1, 2]]
    torch.testing.assert_close(r.top_logp, lp.gather(-1, r.top_ids))
    assert token_logprobs(x, t).top_ids is None


def test_gradients():
    torch.manual_seed(0)
    x = torch.randn(2, 3, 6, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, 6, (2, 3))
    t[0, 0] = -100
    assert torch.autograd.gradcheck(lambda v: token_logprobs(v, t)[:2], (x,))


def test_masked_and_missing():
    inf = float("inf")
    x = torch.tensor([[-inf, -inf, -inf], [0.0, -inf, -inf], [1.0, 2.0, 3.0], [1.0, 2.0, 3.0]])
    x.requires_grad_(True)
    t = torch.tensor([1, 0, -100, 3])
    r = token_logprobs(x, t, top=2)
    assert r.logp.tolist()[:3] == [-inf, 0.0, 0.0] and r.logp[3].isnan()
    assert r.entropy[:2].tolist() == [0.0, 0.0]
    assert r.top_ids[0].tolist() == [0, 1]
    dx, = torch.autograd.grad(r.logp[1:].sum(), x)
    assert (dx[2] == 0).all() and dx[3].isnan().all()
    assert token_logprobs(x, t, ignore_index=0).logp[1] == 0


def test_refusals():
    x = torch.randn(3, 6)
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="last dimension"):
        token_logprobs(torch.tensor(1.0), t)
    with pytest.raises(ValueError, match="last dimension"):
        token_logprobs(torch.randn(3, 0), t)
    with pytest.raises(ValueError, match="shape"):
        token_logprobs(x, t[:2])
    with pytest.raises(ValueError, match="shape"):
        token_logprobs(x, t[:, None])
    with pytest.raises(ValueError, match="whole numbers"):
        token_logprobs(x, t.float())
    for top in (-1, 7):
        with pytest.raises(ValueError, match="top"):
            token_logprobs(x, t, top=top)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(torch.randn(3, 100), t, top=65)
    with pytest.raises(ValueError, match="floating"):
        token_logprobs(x.int(), t)


def test_ignored_index_of_more_than_64_bits():
    """2^64 - 100 would be -100 in the kernels."""
    x, t = torch.randn(3, 5), torch.tensor([0, -100, 4])
    for index in (2 ** 64 - 100, 2 ** 63, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="64-bit"):
            token_logprobs(x, t, ignore_index=index)
    assert token_logprobs(x, t, ignore_index=-2 ** 63).logp[1].isnan()
