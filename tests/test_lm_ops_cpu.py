"""The language-model operators on the CPU path: against 64-bit
definitions, and what they refuse."""
import math

import pytest
import torch

from sparkflow_amd.ops import functional as F

from tests import lm_oracle as oracle

TYPES = [torch.float32, torch.bfloat16, torch.float16]


# -- dropout ------------------------------------------------------------------


def test_philox_known_answers():
    """The published vectors of Philox4x32-10."""
    for state, block, words in (
            ((0, 0), 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
            ((2 ** 64 - 1, 2 ** 64 - 1), 2 ** 64 - 1,
             "408f276d 41c83b0e a20bc7c6 6d5451fd")):
        got = oracle.philox_words(*state, block, 1)
        assert ["%08x" % int(v) for v in got] == words.split()
    got = F._philox_words(F.dropout_state(0), 4)
    assert ["%08x" % int(v) for v in got] == \
        "6627e8d5 e169c58d bc57ac4c 9b00dbd8".split()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (9,), (30, 41), (2, 3, 5)])
def test_dropout(dtype, shape):
    state = F.dropout_state(-3, 2 ** 40 + 1)
    x = torch.randn(*shape).to(dtype).requires_grad_()
    y = F.dropout(x, 0.3, state)
    want = oracle.dropout(x.detach(), state, 0.3)
    tol = want.abs() * (2.01 * oracle.U32 + oracle.half_step(dtype)) + (
        2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((y.detach().double() - want).abs() <= tol).all()
    g = torch.randn(*shape).to(dtype)
    (dx,) = torch.autograd.grad(y, x, g)
    want = oracle.dropout(g, state, 0.3)
    assert torch.equal(dx == 0, want == 0) and dx.dtype == dtype


def test_dropout_share_and_draws():
    state = F.dropout_state(1)
    x = torch.ones(100000)
    first = F.dropout(x, 0.2, F.dropout_next(state))
    second = F.dropout(x, 0.2, F.dropout_next(state))
    assert state.tolist() == [1, 2]
    assert torch.equal(first, F.dropout(x, 0.2, F.dropout_state(1, 0)))
    assert not torch.equal(first, second)
    for y in (first, second):  # within five standard deviations
        share = float((y != 0).float().mean())
        assert abs(share - 0.8) < 5 * math.sqrt(0.16 / 100000)
    both = float(((first != 0) & (second != 0)).float().mean())
    assert abs(both - 0.64) < 5 * math.sqrt(0.64 * 0.36 / 100000)


def test_dropout_saved_state_may_not_change():
    state = F.dropout_state(1)
    x = torch.ones(8, requires_grad=True)
    y = F.dropout(x, 0.5, state)
    F.dropout_next(state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_dropout_edges():
    state = F.dropout_state(1)
    x = torch.tensor([math.inf, math.nan] * 64)
    y = F.dropout(x, 0.5, state)
    assert (y[~oracle.kept(state, 0.5, 128)] == 0).all()
    assert F.dropout(x, 0.0, state) is x
    assert F.dropout(x, 0.5, state, training=False) is x
    assert (F.dropout(x, 1.0, state) == 0).all()
    assert F.dropout(x[:0], 0.5, state).shape == (0,)


def test_dropout_refuses():
    state = F.dropout_state(1)
    x = torch.ones(4)
    for bad in (x.double(), x.long()):
        with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
            F.dropout(bad, 0.5, state)
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="within 0 and 1"):
            F.dropout(x, p, state)
    for bad in (state.int(), state[:1], torch.zeros(4).long()[::2]):
        with pytest.raises(ValueError, match="two contiguous int64"):
            F.dropout(x, 0.5, bad)
        with pytest.raises(ValueError, match="two contiguous int64"):
            F.dropout_next(bad)
    with pytest.raises(ValueError, match="state on meta"):
        F.dropout(x, 0.5, state.to("meta"))


# -- log-probabilities --------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,k", [((1, 1), 1), ((6, 10), 3),
                                     ((5, 40), 32), ((7, 333), 0)])
def test_logprobs(dtype, shape, k):
    m, c = shape
    logits = (torch.randn(m, c) * 3).to(dtype)
    if m > 4:
        logits[0, 1:] = -math.inf
        logits[1] = -math.inf
        logits[2] = torch.finfo(dtype).min
        logits[3, ::2] = logits[3, 0]
    tokens = torch.arange(m) % c
    if m > 5:
        tokens[5] = -100
    x = logits.clone().requires_grad_()
    r = F.token_logprobs(x, tokens, top_k=k)
    logp, h, top, ids = oracle.logprobs(logits, tokens, k)
    assert torch.equal(r.top_ids, ids)
    for got, want, ent in ((r.logp, logp, False), (r.entropy, h, True),
                           (r.top_logp, top, False)):
        off = (got.detach().double() - want).abs()
        off = torch.where(got == want, torch.zeros_like(off), off)
        assert (off <= oracle.logprobs_tol(want, ent, c)).all()
    gs = [torch.randn(m), torch.randn(m), torch.randn(m, k)]
    roots = [r.logp, r.entropy] + ([r.top_logp] if k else [])
    (dx,) = torch.autograd.grad(roots, x, gs[:len(roots)])
    want, tol = oracle.logprobs_grad(logits, tokens, k, gs)
    assert ((dx.double() - want).abs() <= tol).all()


def test_logprobs_agrees_with_softmax_xent():
    logits = torch.randn(12, 10)
    labels = torch.randint(0, 10, (12, 1)).float()  # the engine's labels
    x, y = (logits.clone().requires_grad_() for _ in range(2))
    loss = -F.token_logprobs(x, labels).logp.mean()
    ref = F.softmax_xent(y, labels)
    torch.testing.assert_close(loss, ref)
    loss.backward()
    ref.backward()
    torch.testing.assert_close(x.grad, y.grad)


def test_logprobs_broken_rows_and_tokens():
    logits = torch.randn(5, 9)
    logits[1, 3] = math.nan
    logits[2, 3] = math.inf
    tokens = torch.tensor([9, 0, 0, -1, -100])
    r = F.token_logprobs(logits, tokens, top_k=2)
    assert torch.isnan(r.logp).tolist() == [True] * 4 + [False]
    assert torch.isnan(r.entropy).tolist() == [False, True, True, False,
                                               False]
    assert r.top_ids[[1, 2, 4]].tolist() == [[-1, -1]] * 3


def test_logprobs_refuses():
    x, t = torch.randn(4, 6), torch.zeros(4).long()
    for bad in (x.double(), x.long()):
        with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
            F.token_logprobs(bad, t)
    for bad in (t[:3], t.reshape(2, 2), t.reshape(1, 4)):
        with pytest.raises(ValueError, match="do not fit"):
            F.token_logprobs(x, bad)
    for bad in (t.bool(), t.double(), t.half()):
        with pytest.raises(ValueError, match="whole numbers"):
            F.token_logprobs(x, bad)
    for k in (-1, 7, 33):
        with pytest.raises(ValueError, match="top_k"):
            F.token_logprobs(x, t, top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        F.token_logprobs(torch.randn(4, 60), t, top_k=33)
    with pytest.raises(ValueError, match="classes"):
        F.token_logprobs(x[:, :0], t)
    with pytest.raises(ValueError, match="tokens on meta"):
        F.token_logprobs(x, t.to("meta"))
    y = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(F.token_logprobs(y, t).logp.sum(), y,
                               create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        g.sum().backward()
