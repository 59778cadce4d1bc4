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


def test_logprobs_loss_leaves_ignored_rows_out():
    """The loss of the README: the mean over the rows that are read."""
    logits, labels = torch.randn(12, 10), torch.randint(0, 10, (12,))
    labels[::3] = -100
    x, y = (logits.clone().requires_grad_() for _ in range(2))
    logp = F.token_logprobs(x, labels, ignore_index=-100).logp
    loss = -logp.sum() / (labels != -100).sum()
    ref = torch.nn.functional.cross_entropy(y, labels, ignore_index=-100)
    torch.testing.assert_close(loss, ref)
    loss.backward()
    ref.backward()
    torch.testing.assert_close(x.grad, y.grad)


def check_gradient_of_impossible_classes(device):
    """What flows to a named class reaches its logit, possible or not; the
    others' probabilities are 0 and add nothing."""
    rows = torch.tensor([[0.0, 1.0, -math.inf, -math.inf]] * 2)
    tokens = torch.tensor([2, 0])
    x = rows.to(device).requires_grad_()
    r = F.token_logprobs(x, tokens.to(device), top_k=3)
    assert r.logp.tolist()[0] == -math.inf
    assert r.top_logp[:, 2].tolist() == [-math.inf] * 2
    y = rows.double().requires_grad_()
    logp = torch.log_softmax(y, 1)
    for got, want in ((r.logp, logp.gather(1, tokens.unsqueeze(1))),
                      (r.top_logp, logp.gather(1, r.top_ids.cpu())),
                      (r.top_logp[:, :2], logp[:, :2])):
        (dx,) = torch.autograd.grad(got.sum(), x, retain_graph=True)
        (dy,) = torch.autograd.grad(want.sum(), y, retain_graph=True)
        # four terms of size 3 at most, each a few half steps off
        assert ((dx.cpu().double() - dy).abs() <= 64 * oracle.U32).all()
    (dx,) = torch.autograd.grad(r.entropy.sum(), x)
    assert (dx[:, 2:] == 0).all() and torch.isfinite(dx).all()


def test_logprobs_gradient_of_impossible_classes():
    check_gradient_of_impossible_classes("cpu")


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


# -- low-rank adapters --------------------------------------------------------


def _adapter_inputs(m, k, n, r, e, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen) * std).to(dtype)

    return (normal(m, n), normal(m, k), normal(e, r, k, std=k ** -0.5),
            normal(e, n, r, std=r ** -0.5),
            torch.randint(-1, e, (m,), generator=gen),
            torch.rand(e, generator=gen) + 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (9, 20, 7, 3, 4),
                                   (40, 17, 33, 16, 2), (5, 8, 8, 2, 30)])
def test_adapter_add(dtype, shape):
    base, x, a, b, ids, scale = _adapter_inputs(*shape, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (base, x, a, b)]
    y = F.adapter_add(*leaves, ids, scale=scale)
    g = torch.randn(y.shape).to(dtype)
    grads = torch.autograd.grad(y, leaves, g)
    assert torch.equal(grads[0], g)
    want = oracle.adapter(base, x, a, b, ids, scale, g)
    for got, (value, tol) in zip((y,) + grads[1:], want):
        assert got.dtype == dtype
        assert ((got.detach().double() - value).abs() <= tol).all()


def test_adapter_add_scale_act_groups_and_shapes():
    base, x, a, b, ids, _ = _adapter_inputs(12, 6, 5, 2, 3)
    y = F.adapter_add(base, x, a, b, ids, scale=0.5)
    value, tol = oracle.adapter(base, x, a, b, ids, 0.5)[0]
    assert ((y.double() - value).abs() <= tol).all()
    relu = F.adapter_add(base, x, a, b, ids, scale=0.5, act="relu")
    assert torch.equal(relu, torch.relu(y))
    groups = F.adapter_groups(ids, 3)
    assert torch.equal(F.adapter_add(base, x, a, b, groups, scale=0.5), y)
    shaped = F.adapter_add(base.reshape(3, 4, 5), x.reshape(3, 4, 6), a, b,
                           ids.reshape(3, 4), scale=0.5)
    assert torch.equal(shaped.reshape(12, 5), y)
    none = F.adapter_add(base, x, a, b, torch.full_like(ids, -7))
    assert torch.equal(none, base)
    bad = ids.clone()
    bad[3] = 3
    y = F.adapter_add(base, x, a, b, bad)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[:3]).all()


def test_adapter_add_act_gradient_by_differences():
    base, x, a, b, ids, scale = _adapter_inputs(6, 5, 4, 2, 2, seed=3)
    ids[0], ids[1] = 0, -1
    leaves = [t.clone().requires_grad_() for t in (base, x, a, b)]
    g = torch.randn(6, 4)
    y = F.adapter_add(*leaves, ids, scale=scale, act="sigmoid")
    grads = torch.autograd.grad(y, leaves, g)

    def loss(*ts):
        pre = oracle.adapter(*ts, ids, scale)[0][0]
        return float((torch.sigmoid(pre) * g).sum())

    for w in range(4):
        ts = [t.double() for t in (base, x, a, b)]
        for i in range(ts[w].numel()):
            up, down = (list(ts), list(ts))
            up[w], down[w] = ts[w].clone(), ts[w].clone()
            up[w].view(-1)[i] += 1e-5
            down[w].view(-1)[i] -= 1e-5
            slope = (loss(*up) - loss(*down)) / 2e-5
            assert abs(float(grads[w].reshape(-1)[i]) - slope) < 1e-5


def test_adapter_add_refuses():
    base, x, a, b, ids, scale = _adapter_inputs(4, 6, 5, 2, 3)

    def refused(match, **changed):
        args = dict(base=base, x=x, a=a, b=b, ids=ids)
        args.update(changed)
        with pytest.raises(ValueError, match=match):
            F.adapter_add(**args)

    refused("fp32, bf16 or fp16", base=base.double())
    refused("base is torch.float16", base=base.half())
    refused("b is torch.bfloat16", b=b.bfloat16())
    refused("do not fit", a=a[:2])
    refused("do not fit", b=b[:, :, :1])
    refused("do not fit", a=a[0])
    refused("x .* do not fit", x=x[:, :5])
    refused("x .* do not fit", base=base[:3])
    refused("x .* do not fit", ids=ids[:3])
    refused("integer type", ids=ids.float())
    refused("integer type", ids=ids > 0)
    refused("ids on meta", ids=ids.to("meta"))
    refused("scale must", scale=scale[:2])
    refused("scale must", scale=scale.double())
    refused("no gradient", scale=scale.clone().requires_grad_())
    refused("grouped for 4", ids=F.adapter_groups(ids, 4))
    refused("rank must", a=torch.randn(3, 129, 6), b=torch.randn(3, 5, 129))
    refused("rank must", a=a[:, :0], b=b[:, :, :0])
    refused("within 1 and 1024", a=torch.randn(1025, 1, 6),
            b=torch.randn(1025, 5, 1))
    for e in (0, 1025):
        with pytest.raises(ValueError, match="adapters must be"):
            F.adapter_groups(ids, e)
    with pytest.raises(KeyError):
        F.adapter_add(base, x, a, b, ids, act="tanh")
    refused("activation code", act=3)


# -- modules and models -------------------------------------------------------


def test_dropout_module_with_a_seed():
    from sparkflow_amd import nn as snn

    old, new = snn.Dropout(0.4), snn.Dropout(0.4, seed=7)
    assert list(new.state_dict()) == []  # artifacts of either load as both
    x = torch.ones(4, 50)
    assert torch.equal(new(x), F.dropout(x, 0.4, F.dropout_state(7, 0)))
    assert torch.equal(new(x), F.dropout(x, 0.4, F.dropout_state(7, 1)))
    new.reseed(9, 3)
    assert torch.equal(new(x), F.dropout(x, 0.4, F.dropout_state(9, 3)))
    assert new.eval()(x) is x
    # without a seed: torch's generator, as before
    torch.manual_seed(3)
    want = x * ((torch.rand_like(x) < 0.6).to(x.dtype) / 0.6)
    torch.manual_seed(3)
    assert torch.equal(old(x), want)
    with pytest.raises(ValueError, match="without a seed"):
        old.reseed(1)


def check_dropout_run_again(device):
    """A recomputed forward draws the mask of the state that it is given."""
    from torch.utils.checkpoint import checkpoint

    from sparkflow_amd import nn as snn

    drop = snn.Dropout(0.5, seed=4).to(device)
    x = torch.ones(64, device=device, requires_grad=True)
    masks = []
    for _ in range(2):
        state = F.dropout_next(drop.rng_state)
        y = checkpoint(lambda t: F.dropout(t, drop.p, state) ** 2, x,
                       use_reentrant=False)
        (dx,) = torch.autograd.grad(y.sum(), x)
        assert torch.equal(dx, 2 * y)  # 2 x / (1 - p)^2 = 8 where y is 4
        masks.append(y != 0)
    assert not torch.equal(*masks)
    assert drop.rng_state.tolist() == [4, 2]


def test_dropout_run_again():
    check_dropout_run_again("cpu")


def _seeded_dropout_mlp():
    from sparkflow_amd.models import dropout_mlp

    return dropout_mlp(in_dim=6, hidden=16, p=0.3, seed=5)


def test_seeded_dropout_model_serializes():
    from sparkflow_amd.graph_utils import build_graph
    from sparkflow_amd.models import dropout_mlp
    from sparkflow_amd.utils.serialization import module_from_json

    again = module_from_json(build_graph(_seeded_dropout_mlp))
    assert again.drop.rng_state.tolist() == [5, 0]
    plain = dropout_mlp(in_dim=6, hidden=16)
    assert list(plain.state_dict()) == list(again.state_dict())
    x, y = torch.randn(8, 6), torch.rand(8, 1)
    again.train().compute_loss(again(x), y).backward()
    assert all(torch.isfinite(p.grad).all() for p in again.parameters())


def test_adapter_linear_module():
    from sparkflow_amd import nn as snn
    from sparkflow_amd.utils.serialization import flat_size, param_list

    linear = snn.Linear(12, 7, activation="relu")
    layer = snn.AdapterLinear.from_linear(linear, rank=3, adapters=4,
                                          scale=0.5)
    x = torch.randn(10, 12)
    assert torch.equal(layer(x), linear(x))  # B is zero at first
    assert [id(p) for p in param_list(layer)] == [id(layer.a), id(layer.b)]
    assert flat_size(layer) == 4 * 3 * (12 + 7)
    with torch.no_grad():
        layer.b.normal_()
    ids = torch.tensor([0, 1, 2, 3, -1, 3, 2, 1, 0, -1])
    base = F.linear_act(x, linear.weight, linear.bias)
    value, tol = oracle.adapter(base.detach(), x, layer.a, layer.b, ids,
                                0.5)[0]
    got = layer(x, ids)
    assert ((got.double() - torch.relu(value)).abs() <= tol).all()
    assert torch.equal(layer(x, F.adapter_groups(ids, 4)), got)
    x.requires_grad_()
    layer(x, ids).sum().backward()
    assert layer.weight.grad is None and layer.bias.grad is None
    assert layer.a.grad is not None and x.grad is not None


def test_adapter_linear_rows_of_any_shape():
    from sparkflow_amd import nn as snn

    layer = snn.AdapterLinear(6, 4, 2, adapters=3, activation="relu")
    with torch.no_grad():
        layer.b.normal_()
    x, ids = torch.randn(2, 5, 6), torch.arange(10).reshape(2, 5) % 4 - 1
    want = layer(x.reshape(10, 6), ids.reshape(10))
    for leaf in (x.clone(), x.transpose(1, 2).contiguous().transpose(1, 2)):
        leaf.requires_grad_()
        got = layer(leaf, ids)
        torch.testing.assert_close(got, want.reshape(2, 5, 4))
        got.sum().backward()
        assert leaf.grad.shape == x.shape
    torch.testing.assert_close(layer(x[1, 2]), layer(x[:, 2])[1])
    assert layer(x[:0]).shape == (0, 5, 4)


def test_frozen_linear_gradient_of_x():
    for act in ("none", "relu", "sigmoid"):
        x, w, b = torch.randn(5, 6), torch.randn(6, 4), torch.randn(4)
        one = x.clone().requires_grad_()
        F.linear_act(one, w, b, act).sum().backward()
        two, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
        F.linear_act(two, w2, b, act).sum().backward()
        torch.testing.assert_close(one.grad, two.grad)


def test_classifier_score():
    from sparkflow_amd.models import mnist_mlp

    model = mnist_mlp()
    x, labels = torch.randn(5, 784), torch.tensor([3, 1, 4, 1, 5])
    r = model.score(x, labels.float().unsqueeze(1), top_k=2)
    logp = torch.log_softmax(model(x), 1)
    torch.testing.assert_close(r.logp, logp[torch.arange(5), labels])
    assert torch.equal(r.top_ids[:, 0].float(), model.predict(x))


class _AdaptedClassifier(torch.nn.Module):
    """Fine-tuning as a user writes it: dropout on the input of adapters
    beside frozen layers, against the log-probabilities of the answers and
    a reward for entropy."""

    def __init__(self, dims, rank, adapters, seed):
        super().__init__()
        from sparkflow_amd import nn as snn

        self.drop = snn.Dropout(0.2, seed=seed)
        self.hidden = snn.AdapterLinear(dims[0], dims[1], rank, adapters,
                                        activation="relu")
        self.out = snn.AdapterLinear(dims[1], dims[2], rank, adapters)

    def forward(self, x, ids=None):
        return self.out(self.hidden(self.drop(x), ids), ids)

    def compute_loss(self, out, target):
        r = F.token_logprobs(out, target)
        return -(r.logp + 0.01 * r.entropy).mean()


def check_operators_together(device, rows=20):
    """Dropout, adapters and log-probabilities in one training step, against
    autograd over plain operations in 64 bits."""
    torch.manual_seed(0)
    model = _AdaptedClassifier([12, 9, 6], 2, 3, seed=11)
    with torch.no_grad():
        for p in (model.hidden.b, model.out.b):
            p.normal_(std=0.3)
    x, ids = torch.randn(rows, 12), torch.randint(-1, 3, (rows,))
    y = torch.randint(0, 6, (rows,))
    y[4] = -100
    model.to(device)
    loss = model.compute_loss(
        model(x.to(device), F.adapter_groups(ids.to(device), 3)),
        y.to(device))
    loss.backward()

    keep = oracle.kept(F.dropout_state(11), 0.2, x.numel()).reshape(x.shape)
    leaves = {n: p.detach().cpu().double().requires_grad_()
              for n, p in model.named_parameters()}
    h = x.double() * keep / 0.8
    mine = (ids.unsqueeze(1) == torch.arange(3)).double()
    for layer in ("hidden", "out"):
        w, bias, a, b = (leaves["%s.%s" % (layer, n)]
                         for n in ("weight", "bias", "a", "b"))
        z = torch.einsum("mk,erk->mer", h, a) * mine.unsqueeze(2)
        h = h @ w + bias + torch.einsum("mer,enr->mn", z, b)
        if layer == "hidden":
            h = torch.relu(h)
    logp = torch.log_softmax(h, 1)
    live = y != -100
    chosen = logp[torch.arange(rows), y.clamp(min=0)] * live
    entropy = -(logp.exp() * logp).sum(1) * live
    want = -(chosen + 0.01 * entropy).mean()
    want.backward()
    torch.testing.assert_close(loss.cpu().double(), want, rtol=1e-5,
                               atol=1e-6)
    for n, p in model.named_parameters():
        if p.requires_grad:
            torch.testing.assert_close(p.grad.cpu().double(),
                                       leaves[n].grad, rtol=1e-4, atol=1e-6)


def test_operators_together():
    check_operators_together("cpu")


def _adapted_builder():
    from tests.test_lm_ops_cpu import _AdaptedClassifier

    torch.manual_seed(1)
    return _AdaptedClassifier([10, 16, 4], 2, 1, seed=3)


def test_adapters_train_through_the_engine():
    import numpy as np

    from sparkflow_amd.graph_utils import build_graph
    from sparkflow_amd.parallel.ps import OptimizerSpec, PSCore, TrainConfig
    from sparkflow_amd.parallel.transport import LocalTransport
    from sparkflow_amd.parallel.worker import Worker

    graph_json = build_graph(_adapted_builder)
    ps = PSCore(graph_json, OptimizerSpec("adam", 0.01), device="cpu")
    before = ps.weights.clone()
    assert before.numel() == 2 * (10 + 16) + 2 * (16 + 4)
    worker = Worker(graph_json, LocalTransport(ps, "cpu"),
                    TrainConfig(iters=3, mini_batch=8,
                                mini_stochastic_iters=1, seed=0),
                    device="cpu")
    frozen = worker.module.hidden.weight.clone()
    rng = np.random.default_rng(0)
    worker.run(rng.random((24, 10), dtype=np.float32),
               rng.integers(0, 4, (24, 1)).astype(np.float32))
    assert ps.update_count == 3
    assert torch.isfinite(ps.weights).all()
    assert not torch.equal(ps.weights, before)
    assert torch.equal(worker.module.hidden.weight, frozen)
