"""The language-model operators on the GPU against 64-bit definitions:
dropout from a counter, token log-probabilities, low-rank adapters."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from sparkflow_amd import ops
    from sparkflow_amd.ops import functional as F
else:
    pytest.skip("no GPU in this container", allow_module_level=True)

from tests import lm_oracle as oracle  # noqa: E402

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def setup_module():
    assert ops.available(), f"extension missing: {ops.loader.LAST_ERROR}"


def _randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)


def _within(got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    assert not torch.isnan(off).any(), "NaN where there should be none"
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(off)
    worst = (off - tol).max() if off.numel() else 0.0
    assert worst <= 0, f"{float(worst)} over a bound of {float(tol.max())}"


# -- dropout ------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (7,), (8,), (9,), (63, 33),
                                   (1023, 1001), (2, 3, 4, 5), (300, 256)])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.977])
def test_dropout_values(dtype, shape, p):
    x = _randn(*shape, dtype=dtype, seed=1).requires_grad_()
    state = F.dropout_state(-7, 2 ** 33 + 5, device=DEV)
    y = F.dropout(x, p, state)
    want = oracle.dropout(x.detach(), state, p)
    # the scale is rounded once, the product once to 32 bits, then to dtype
    tol = want.abs() * (2.01 * oracle.U32 + oracle.half_step(dtype))
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    _within(y, want, tol)
    assert torch.equal(y.detach().cpu() == 0, (want == 0))
    # the same bits as the CPU path
    cpu = F.dropout(x.detach().cpu(), p, state.cpu())
    assert torch.equal(y.detach().cpu(), cpu)
    g = _randn(*shape, dtype=dtype, seed=2)
    (dx,) = torch.autograd.grad(y, x, g)
    assert torch.equal(dx.cpu(), F.dropout(g.cpu(), p, state.cpu()))


@pytest.mark.parametrize("n", [256 * 256 * 8 * 4 + 3, 256 * 256 * 8 * 8 + 9])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_large_and_small_launch_agree(n, dtype):
    x = _randn(n, dtype=dtype, seed=3)
    state = F.dropout_state(11, device=DEV)
    y = F.dropout(x, 0.25, state)
    part = 4 * 1001
    assert torch.equal(y[:part], F.dropout(x[:part], 0.25, state))
    keep = oracle.kept(state, 0.25, 4003, first=n // 4 * 4 - 4000)
    tail = y[n // 4 * 4 - 4000:].cpu()
    assert torch.equal(tail != 0, keep[:len(tail)] & (
        x[n // 4 * 4 - 4000:].cpu() != 0))


def test_dropout_index_past_32_bits():
    n = 2 ** 32 + 2 ** 10 + 3
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    state = F.dropout_state(5, 6, device=DEV)
    y = F.dropout(x, 0.5, state)
    for first in (0, 2 ** 31 - 64, 2 ** 32 - 64, n // 4 * 4 - 256):
        m = min(259, n - first)
        assert torch.equal(y[first:first + m].cpu() == 2,
                           oracle.kept(state, 0.5, m, first=first))


def test_dropout_drops_infinities_and_edges_of_p():
    state = F.dropout_state(1, device=DEV)
    x = torch.full((4096,), math.inf, device=DEV)
    x[1::2] = math.nan
    y = F.dropout(x, 0.5, state)
    keep = oracle.kept(state, 0.5, 4096).to(DEV)
    assert (y[~keep] == 0).all()
    assert not torch.isfinite(y[keep]).any()
    assert F.dropout(x, 0.0, state) is x
    assert F.dropout(x, 0.5, state, training=False) is x
    assert (F.dropout(x, 1.0, state) == 0).all()
    small = F.dropout(torch.ones(64, device=DEV), 2.0 ** -40, state)
    assert (small == 1).all()
    assert F.dropout(x[:0], 0.5, state).shape == (0,)
    assert F.dropout(x[0], 0.5, state).shape == ()


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_views(dtype):
    state = F.dropout_state(9, device=DEV)
    big = _randn(70, 67, dtype=dtype, seed=4)
    for view in (big[1:, 3:], big.t(), big[:, ::2], big.reshape(-1)[1:],
                 big[:1].expand(5, 67)):
        got = F.dropout(view, 0.4, state)
        assert torch.equal(got.cpu(),
                           F.dropout(view.cpu().contiguous(), 0.4,
                                     state.cpu()))
    x = big[1:, 3:].detach().requires_grad_()
    g = _randn(67, 70 - 1 + 0, dtype=dtype, seed=5)[3:].t()
    y = F.dropout(x, 0.4, state)
    (dx,) = torch.autograd.grad(y, x, g)
    assert torch.equal(dx.cpu(),
                       F.dropout(g.cpu().contiguous(), 0.4, state.cpu()))


def test_dropout_twice_differentiable():
    state = F.dropout_state(2, device=DEV)
    x = _randn(33, 5).requires_grad_()
    g = _randn(33, 5, seed=1).requires_grad_()
    y = F.dropout(x, 0.3, state)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    (dg,) = torch.autograd.grad(dx, g, torch.ones_like(dx))
    assert torch.equal(dg, F.dropout(torch.ones_like(dx), 0.3, state))


def test_dropout_state_steps_and_captures():
    state = F.dropout_state(2 ** 63 + 1, 2 ** 64 - 2, device=DEV)
    x = torch.ones(1000, device=DEV)

    def step():
        return F.dropout(x, 0.5, F.dropout_next(state))

    for _ in range(2):
        step()  # the counter passes 2^64
    assert state.tolist()[1] == 0
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    masks = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        masks.append(y.clone())
        eager = F.dropout(x, 0.5, F.dropout_state(2 ** 63 + 1, 1 + i,
                                                  device=DEV))
        assert torch.equal(masks[-1], eager)
        x.mul_(1.0)  # the program's own work between replays
    assert not torch.equal(masks[0], masks[1])
    assert state.tolist()[1] == 5


def test_dropout_on_another_stream():
    state = F.dropout_state(3, device=DEV)
    x = _randn(100000)
    want = F.dropout(x, 0.2, state)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = F.dropout(x, 0.2, state)
    side.synchronize()
    assert torch.equal(got, want)


# -- log-probabilities --------------------------------------------------------


def _check_logprobs(logits, tokens, k, ignore=-100, grads=(1, 1, 1)):
    x = logits.detach().requires_grad_()
    m, c = x.shape
    r = F.token_logprobs(x, tokens, top_k=k, ignore_index=ignore)
    logp, h, top, ids = oracle.logprobs(logits, tokens, k, ignore)
    assert torch.equal(r.top_ids.cpu(), ids)
    _within(r.logp, logp, oracle.logprobs_tol(logp, False, c))
    _within(r.entropy, h, oracle.logprobs_tol(h, True, c))
    _within(r.top_logp, top, oracle.logprobs_tol(top, False, c))
    gs = [_randn(m, seed=21), _randn(m, seed=22), _randn(m, k, seed=23)]
    roots = [r.logp, r.entropy, r.top_logp]
    use = [i for i in range(3) if grads[i] and (i < 2 or k)]
    (dx,) = torch.autograd.grad([roots[i] for i in use], x,
                                [gs[i] for i in use])
    want, tol = oracle.logprobs_grad(
        logits, tokens, k, [gs[i] if i in use else None for i in range(3)],
        ignore)
    assert dx.dtype == logits.dtype
    _within(dx, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,k", [
    ((1, 1), 1), ((1, 2), 0), ((3, 7), 7), ((300, 10), 3), ((5, 64), 32),
    ((4, 65), 5), ((9, 513), 20), ((2, 1025), 32), ((7, 2047), 1),
    ((3, 4096), 20), ((2, 8200), 32), ((1, 50001), 20), ((2, 131072), 5),
    ((520, 4103), 3)])
def test_logprobs_values(dtype, shape, k):
    m, c = shape
    logits = _randn(m, c, dtype=dtype, seed=7, std=3.0)
    gen = torch.Generator().manual_seed(8)
    tokens = torch.randint(0, c, (m,), generator=gen).to(DEV)
    if m > 2:
        tokens[1] = -100
    _check_logprobs(logits, tokens, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [40, 700, 5000, 20000])
def test_logprobs_masks(dtype, c):
    logits = _randn(8, c, dtype=dtype, seed=9, std=4.0)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf                       # nothing is possible
    logits[1, 1:] = -math.inf                   # one class is
    logits[2, ::2] = low                        # masked by the lowest value
    logits[3] = low                             # ... everywhere
    logits[4, : c // 2] = -math.inf             # half of them
    logits[5] = 0.5                             # all equal
    logits[6, 5:] = -math.inf                   # fewer than top_k
    tokens = torch.tensor([3, 0, 1, 2, 0, c - 1, 9, 4], device=DEV)
    _check_logprobs(logits, tokens, 20)
    _check_logprobs(logits, tokens, 0)


@pytest.mark.parametrize("grads", [(1, 0, 0), (0, 1, 0), (0, 0, 1),
                                   (1, 0, 1)])
def test_logprobs_single_gradients(grads):
    logits = _randn(6, 999, seed=10, std=2.0)
    tokens = torch.tensor([0, 998, -100, 5, 6, 7], device=DEV)
    _check_logprobs(logits, tokens, 4, grads=grads)


def test_logprobs_ties_and_zeros():
    logits = torch.zeros(3, 6000, device=DEV)
    logits[0, 1::2] = -0.0
    logits[1] = (torch.arange(6000, device=DEV) % 3).float()
    logits[2] = -torch.arange(6000, device=DEV).float().div(1000).floor()
    ids = F.token_logprobs(logits, torch.zeros(3, device=DEV),
                           top_k=32).top_ids.cpu()
    assert ids[0].tolist() == list(range(32))
    assert ids[1].tolist() == [2 + 3 * i for i in range(32)]
    assert ids[2].tolist() == list(range(32))


@pytest.mark.parametrize("dtype,c,rows", [
    (torch.float32, 262144, 512), (torch.bfloat16, 262144, 512),
    (torch.float32, 1000, 4)])
def test_logprobs_large_values_side_by_side(dtype, c, rows):
    """The best classes all in one thread's vectors: more candidates than
    its list holds."""
    n = 16 // torch.finfo(dtype).bits * 8
    nt = 256 if c > 4096 else 64
    at = torch.arange(c, device=DEV)
    logits = torch.zeros(rows, c, dtype=dtype, device=DEV)
    logits[:] = _randn(1, c, dtype=dtype, seed=11)
    hit = at // n % nt == 3
    logits[2, hit] = 10 + _randn(int(hit.sum()), dtype=dtype, seed=12)
    r = F.token_logprobs(logits, torch.zeros(rows, device=DEV), top_k=32)
    for i in (0, 2, rows - 1):
        row = logits[i].double().cpu().numpy()
        want = np.lexsort((np.arange(c), -row))[:32]
        assert r.top_ids[i].tolist() == want.tolist()


def test_logprobs_broken_rows_and_tokens():
    for c in (33, 5000, 30000):
        logits = _randn(6, c, seed=13)
        logits[1, c // 2] = math.nan
        logits[2, 7] = math.inf
        logits[3, :] = -math.inf
        logits[3, c - 1] = math.nan
        tokens = torch.tensor([c, 2, 3, 4, -1, -100], device=DEV)
        x = logits.requires_grad_()
        r = F.token_logprobs(x, tokens, top_k=5)
        assert torch.isnan(r.logp[:5]).all() and r.logp[5] == 0
        assert torch.isnan(r.entropy).tolist() == [False, True, True, True,
                                                   False, False]
        assert torch.isnan(r.top_logp[1:4]).all()
        assert (r.top_ids[1:4] == -1).all() and (r.top_ids[5] == -1).all()
        assert (r.top_ids[[0, 4]] >= 0).all()
        (dx,) = torch.autograd.grad(r.logp.sum(), x, retain_graph=True)
        assert torch.isnan(dx[:5]).all() and (dx[5] == 0).all()
        (dx,) = torch.autograd.grad(r.entropy.sum(), x)
        assert torch.isfinite(dx[[0, 4, 5]]).all()
        cpu = F.token_logprobs(x.detach().cpu(), tokens.cpu(), top_k=5)
        assert torch.equal(cpu.top_ids, r.top_ids.cpu())
        for got, want in zip(r[:3], cpu[:3]):
            torch.testing.assert_close(got.detach().cpu(), want,
                                       equal_nan=True, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_layouts(dtype):
    pad = _randn(4, 6, 1100, dtype=dtype, seed=14, std=2.0)
    tokens = torch.arange(24, device=DEV).reshape(4, 6)
    views = [pad[..., :1001], pad[..., 3:1004], pad[:, ::2, 1:1000],
             pad[:1, :1, :1001].expand(4, 6, 1001),
             pad[..., :999].transpose(0, 1).contiguous().transpose(0, 1),
             pad[..., :1].expand(4, 6, 50)]
    for view in views:
        t = tokens[:, :view.shape[1]]
        leaf = view.detach().requires_grad_()
        got = F.token_logprobs(leaf, t, top_k=3)
        flat = view.detach().contiguous().requires_grad_()
        want = F.token_logprobs(flat, t, top_k=3)
        for a, b in zip(got, want):
            assert a.shape[:2] == t.shape and torch.equal(a, b)
        (da,) = torch.autograd.grad(got.logp.sum(), leaf)
        (db,) = torch.autograd.grad(want.logp.sum(), flat)
        assert torch.equal(da, db)
    one = F.token_logprobs(pad[0, 0], torch.tensor(5, device=DEV), top_k=2)
    assert one.logp.shape == () and one.top_ids.shape == (2,)
    base = pad[0, 0].float().requires_grad_()
    rows = base.unsqueeze(0).expand(3, 1100)  # the gradient of a broadcast
    r = F.token_logprobs(rows, torch.tensor([1, 2, 3], device=DEV))
    (d,) = torch.autograd.grad(r.logp.sum(), base)
    each = base.detach().repeat(3, 1).requires_grad_()
    r = F.token_logprobs(each, torch.tensor([1, 2, 3], device=DEV))
    (e,) = torch.autograd.grad(r.logp.sum(), each)
    torch.testing.assert_close(d, e.sum(0), rtol=1e-5, atol=1e-6)


def test_logprobs_token_types():
    logits = _randn(5, 77, seed=15)
    tokens = torch.tensor([0, 76, -100, 3, 4], device=DEV)
    want = F.token_logprobs(logits, tokens)
    for t in (tokens.float(), tokens.int(), tokens.unsqueeze(1),
              tokens.float().unsqueeze(1), tokens.to(torch.int16)):
        assert torch.equal(F.token_logprobs(logits, t).logp, want.logp)
    other = F.token_logprobs(logits, tokens, ignore_index=76)
    assert other.logp[1] == 0 and torch.isnan(other.logp[2])


def test_logprobs_no_rows():
    x = torch.empty(0, 50, device=DEV, requires_grad=True)
    r = F.token_logprobs(x, torch.empty(0, dtype=torch.int64, device=DEV),
                         top_k=4)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 4)
    r.logp.sum().backward()
    assert x.grad.shape == (0, 50)


def test_logprobs_offsets_past_32_bits():
    m, c = 40000, 60001
    logits = torch.empty(m, c, dtype=torch.bfloat16, device=DEV)
    logits.normal_(0, 2, generator=torch.Generator(DEV).manual_seed(3))
    tokens = torch.arange(m, device=DEV)
    x = logits.requires_grad_()
    r = F.token_logprobs(x, tokens, top_k=2)
    (dx,) = torch.autograd.grad(r.logp.sum(), x)
    for at in (0, 35791, m - 1):
        row, t = logits[at:at + 1].detach(), tokens[at:at + 1]
        logp, h, top, ids = oracle.logprobs(row, t, 2)
        assert torch.equal(r.top_ids[at:at + 1].cpu(), ids)
        _within(r.logp[at:at + 1], logp, oracle.logprobs_tol(logp, False, c))
        want, tol = oracle.logprobs_grad(
            row, t, 2, [torch.ones(1), None, None])
        _within(dx[at:at + 1], want, tol)


def test_logprobs_gradient_by_differences():
    logits = _randn(3, 11, seed=16)
    tokens = torch.tensor([4, 10, 0], device=DEV)

    def loss(x):  # in 64 bits, from the definition
        logp, h, top, _ = oracle.logprobs(x, tokens, 3)
        return float((logp * 2 + h * 0.5 + top.sum(1) * 0.25).sum())

    x = logits.clone().requires_grad_()
    r = F.token_logprobs(x, tokens, top_k=3)
    (r.logp * 2 + r.entropy * 0.5 + r.top_logp.sum(1) * 0.25).sum() \
        .backward()
    base = logits.double().cpu()
    for i in range(3):
        for j in range(11):
            up, down = base.clone(), base.clone()
            up[i, j] += 1e-5
            down[i, j] -= 1e-5
            slope = (loss(up) - loss(down)) / 2e-5
            assert abs(float(x.grad[i, j]) - slope) < 1e-5


def test_logprobs_captured():
    logits = _randn(16, 9001, dtype=torch.bfloat16, seed=17)
    x = logits.clone().requires_grad_()
    tokens = torch.arange(16, device=DEV)
    g = _randn(16, seed=18)

    def step():
        r = F.token_logprobs(x, tokens, top_k=4)
        (d,) = torch.autograd.grad([r.logp, r.entropy], x, [g, g])
        return r.logp.detach(), r.entropy.detach(), r.top_ids, d

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(logits * (1 + i))
        tokens.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
