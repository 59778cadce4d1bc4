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


def test_dropout_run_again_gpu():
    from tests.test_lm_ops_cpu import check_dropout_run_again

    check_dropout_run_again(DEV)


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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [300, 5000, 50001])
def test_logprobs_masked_stretch(dtype, c):
    """Threads, and whole splits, that hold nothing but the lowest value."""
    logits = _randn(6, c, dtype=dtype, seed=14, std=4.0)
    low = torch.finfo(dtype).min
    logits[0, c // 3:] = low
    logits[1, : c - 2] = low
    logits[2, 40:] = low
    logits[3, 1:] = -low         # one far below the others
    logits[4, 7:] = low
    logits[4, :7] = -math.inf
    logits[5, c // 2:] = low / 2
    tokens = torch.tensor([3, c - 1, 39, 2, 9, 1], device=DEV)
    _check_logprobs(logits, tokens, 20)
    _check_logprobs(logits, tokens, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e6, -1e9, -1e10, -1e15, -1e20, -1e30,
                                  -1e37, 1e10, 1e30])
@pytest.mark.parametrize("c", [48, 700, 5000, 50001])
def test_logprobs_masks_of_any_size(dtype, mask, c):
    """Finite masks between common logits and the type's lowest value."""
    logits = _randn(9, c, dtype=dtype, seed=24, std=4.0)
    n = 16 // dtype.itemsize
    logits[0, n:2 * n] = mask               # all that one thread sees
    logits[1, c // 3:] = mask
    logits[2, : c - 2] = mask
    logits[3] = mask
    logits[4, ::2] = mask
    logits[5, : c // 2] = -math.inf         # nothing else is possible
    logits[5, c // 2:] = mask
    logits[6, : c // 2] = torch.finfo(dtype).min
    logits[6, c // 2:] = mask
    logits[7, : c // 2] = 2 * mask          # one mask upon another
    logits[7, c // 2:] = mask
    logits[8, : c // 2] = mask
    tokens = torch.tensor([0, 1, c - 1, 2, 3, c - 1, c - 2, c - 3, 5],
                          device=DEV)
    _check_logprobs(logits, tokens, 20)
    _check_logprobs(logits, tokens, 0)


@pytest.mark.parametrize("at", [2.0 ** 18, 2.0 ** 20, 2.0 ** 21, 2.0 ** 23,
                                2.0 ** 24, 1e9, 1e12])
@pytest.mark.parametrize("c", [1000, 20000])
def test_logprobs_far_from_zero(c, at):
    """Maxima that rise and fall about sizes where fp32 has few places, or
    none, behind the point; rows long enough for several rounds a thread."""
    ramp = torch.linspace(-4, 4, c, device=DEV)
    logits = torch.zeros(512, c, device=DEV)
    rows = [at + ramp, at - ramp, ramp - at, -ramp - at, ramp * at,
            -ramp * at, ramp * (at / 4) - 2.0 ** 20]
    for i, row in enumerate(rows):
        logits[70 * i] = row
    tokens = torch.full((512,), -100, device=DEV)
    tokens[:70 * len(rows):70] = torch.arange(len(rows), device=DEV) + c // 2
    _check_logprobs(logits, tokens, 5)


@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_one_likely_class(dtype):
    """No log-probability is above 0 and no entropy below."""
    value = torch.linspace(-9, 9, 600, device=DEV)
    tokens = torch.zeros(600, device=DEV)
    for c in (1, 3, 64, 1000, 5000):
        for rest in (-math.inf, -300.0):
            logits = torch.full((600, c), rest, device=DEV)
            logits[:, 0] = value
            r = F.token_logprobs(logits.to(dtype), tokens, top_k=1)
            for t in (r.logp, r.top_logp):
                assert (t <= 0).all()
                assert (t >= -oracle.logprobs_tol(
                    torch.zeros(()), False, c)).all()
            assert (r.entropy >= 0).all()
            assert (r.entropy <= oracle.logprobs_tol(
                torch.zeros(()), True, c)).all()


@pytest.mark.parametrize("grads", [(1, 0, 0), (0, 1, 0), (0, 0, 1),
                                   (1, 0, 1)])
def test_logprobs_single_gradients(grads):
    logits = _randn(6, 999, seed=10, std=2.0)
    tokens = torch.tensor([0, 998, -100, 5, 6, 7], device=DEV)
    _check_logprobs(logits, tokens, 4, grads=grads)


def test_logprobs_gradient_of_impossible_classes_gpu():
    from tests.test_lm_ops_cpu import check_gradient_of_impossible_classes

    check_gradient_of_impossible_classes(DEV)


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


def test_logprobs_labels_that_are_no_numbers():
    """fp32 labels of NaN or an infinity name no class."""
    logits = _randn(4, 9, seed=19)
    labels = torch.tensor([math.nan, math.inf, -math.inf, 2.0], device=DEV)
    r = F.token_logprobs(logits, labels, top_k=2)
    assert torch.isnan(r.logp).tolist() == [True, True, True, False]
    assert torch.isfinite(r.entropy).all() and (r.top_ids >= 0).all()
    cpu = F.token_logprobs(logits.cpu(), labels.cpu(), top_k=2)
    assert torch.isnan(cpu.logp).tolist() == [True, True, True, False]


def test_more_rows_than_a_launch_has_are_refused():
    """One row in memory, seen 2^26 times."""
    m = 2 ** 26
    ids = torch.zeros(m, dtype=torch.int64, device=DEV)
    x = torch.zeros(1, 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="too many rows"):
        F.token_logprobs(x.expand(m, 4), ids)
    a = torch.zeros(2, 1, 4, dtype=torch.bfloat16, device=DEV)
    b = torch.zeros(2, 4, 1, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="less than 2\\^26"):
        F.adapter_add(x.expand(m, 4), x.expand(m, 4), a, b, ids)


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


# -- low-rank adapters --------------------------------------------------------


def _adapter_inputs(m, k, n, r, e, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed + 100)
    ids = torch.randint(-1, e, (m,), generator=gen).to(DEV)
    scale = (torch.rand(e, generator=gen) + 0.5).to(DEV)
    return (_randn(m, n, dtype=dtype, seed=seed),
            _randn(m, k, dtype=dtype, seed=seed + 1),
            _randn(e, r, k, dtype=dtype, seed=seed + 2, std=k ** -0.5),
            _randn(e, n, r, dtype=dtype, seed=seed + 3, std=r ** -0.5),
            ids, scale)


def _check_adapter(base, x, a, b, ids, scale, seed=50):
    leaves = [t.detach().requires_grad_() for t in (base, x, a, b)]
    y = F.adapter_add(*leaves, ids, scale=scale)
    g = _randn(*y.shape, dtype=x.dtype, seed=seed)
    grads = torch.autograd.grad(y, leaves, g)
    assert torch.equal(grads[0], g)
    want = oracle.adapter(base, x, a, b, ids, scale, g)
    for got, (value, tol) in zip((y,) + grads[1:], want):
        assert got.dtype == x.dtype and got.is_contiguous()
        _within(got, value, tol)
    return y, grads


@pytest.mark.parametrize("m,e", [(65, 1), (80, 3), (300, 4), (1000, 1024),
                                 (4097, 5), (40000, 300), (8192, 8),
                                 (8193, 640)])
def test_adapter_plan(m, e):
    gen = torch.Generator().manual_seed(m)
    ids = torch.randint(-2, e + 2, (m,), generator=gen)
    plan = ops.hip.adapter_plan(ids.to(DEV), e).cpu()
    group = torch.where(ids < 0, e, torch.where(ids >= e, e + 1, ids))
    counts = torch.bincount(group, minlength=e + 2).tolist()
    starts = [0] + torch.tensor(counts).cumsum(0).tolist()
    sizes = []
    for rows in (16, 64):  # tiles and blocks
        most = m // rows + min(e + 2, m)
        table, plan = plan[:4 * most].reshape(most, 4), plan[4 * most:]
        want = [[g, starts[g] + at, min(rows, counts[g] - at), 0]
                for g in range(e + 2) for at in range(0, counts[g], rows)]
        assert table[:len(want)].tolist() == want
        assert (table[len(want):, 0] == -1).all()
        sizes.append([-(-c // rows) for c in counts])
    perm, seg, tbase = plan.split([m, e + 3, e + 3])
    assert torch.equal(perm.long(), torch.sort(group, stable=True)[1])
    assert seg.tolist() == starts
    assert tbase.tolist() == [0] + torch.tensor(sizes[0]).cumsum(0).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [
    # rows, inputs, outputs, rank, adapters
    (1, 1, 1, 1, 1), (1, 64, 64, 16, 4), (3, 8, 8, 2, 2), (16, 32, 32, 16, 1),
    (17, 33, 65, 7, 3), (32, 512, 384, 16, 64), (33, 100, 31, 17, 2),
    (50, 257, 129, 33, 5), (64, 96, 200, 64, 3), (70, 130, 70, 65, 2),
    (40, 64, 48, 128, 2), (300, 784, 256, 8, 4), (777, 1000, 513, 12, 17),
    (1025, 40, 24, 5, 3), (2500, 200, 136, 20, 3), (1500, 64, 72, 100, 40)])
def test_adapter_values(dtype, shape):
    _check_adapter(*_adapter_inputs(*shape, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [
    (1, 2048, 64, 16, 1), (7, 20000, 40, 128, 3), (32, 4096, 300, 16, 64),
    (33, 2500, 129, 12, 5), (64, 4097, 100, 33, 4), (50, 3333, 71, 64, 2)])
def test_adapter_split_along_inputs(dtype, shape):
    """Up to 64 rows without gradients: several blocks along the inputs."""
    base, x, a, b, ids, scale = _adapter_inputs(*shape, dtype=dtype)
    ids[0] = 0
    value, tol = oracle.adapter(base, x, a, b, ids, scale)[0]
    bad = ids.clone()
    bad[-1] = shape[-1]  # names no adapter
    with torch.no_grad():
        y = F.adapter_add(base, x, a, b, ids, scale=scale)
        _within(y, value, tol)
        relu = F.adapter_add(base, x, a, b, ids, scale=scale, act="relu")
        assert torch.equal(relu, torch.relu(y))
        y2 = F.adapter_add(base, x, a, b, bad, scale=scale)
        assert torch.isnan(y2[-1]).all() and torch.equal(y2[:-1], y[:-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [
    (4096, 136, 72, 32, 3), (4100, 200, 130, 20, 7), (5000, 600, 40, 64, 2),
    (4097, 33, 65, 17, 40)])
def test_adapter_two_tiles_a_block(dtype, shape):
    """From 4096 rows on at ranks of 17 to 64."""
    _check_adapter(*_adapter_inputs(*shape, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(8200, 800, 136, 20, 3),
                                   (8192, 130, 1000, 5, 1),
                                   (20000, 900, 24, 16, 9)])
def test_adapter_long_stretches(dtype, shape):
    """The weights' gradients from more than four tiles a block."""
    _check_adapter(*_adapter_inputs(*shape, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [60, 2000])
@pytest.mark.parametrize("ids", ["none", "one", "last", "runs", "absent"])
def test_adapter_orders(dtype, m, ids):
    base, x, a, b, _, scale = _adapter_inputs(m, 72, 50, 9, 6, dtype=dtype)
    at = torch.arange(m, device=DEV)
    chosen = {"none": torch.full_like(at, -1), "one": torch.zeros_like(at),
              "last": torch.full_like(at, 5), "runs": at * 7 // m - 1,
              "absent": at % 2 * 3}[ids]
    y, grads = _check_adapter(base, x, a, b, chosen, scale)
    for e in range(6):
        if not (chosen == e).any():
            assert (grads[2][e] == 0).all() and (grads[3][e] == 0).all()
    if ids == "none":
        assert torch.equal(y, base) and (grads[1] == 0).all()


def test_adapter_unknown_ids_give_nan():
    for act in ("none", "relu", "sigmoid"):
        base, x, a, b, ids, scale = _adapter_inputs(40, 30, 20, 4, 3)
        bad = ids.clone()
        bad[7], bad[30] = 3, 2 ** 40
        x.requires_grad_()
        y = F.adapter_add(base, x, a, b, bad, scale=scale, act=act)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        ok = torch.ones(40, dtype=torch.bool, device=DEV)
        ok[[7, 30]] = False
        assert torch.isnan(y[~ok]).all() and torch.isnan(dx[~ok]).all()
        want = F.adapter_add(base, x, a, b, ids, scale=scale, act=act)
        assert torch.equal(y[ok], want[ok])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "sigmoid"])
def test_adapter_act(dtype, act):
    base, x, a, b, ids, scale = _adapter_inputs(200, 90, 77, 6, 4,
                                                dtype=dtype)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    y = F.adapter_add(*leaves, ids, scale=0.25, act=act)
    g = _randn(200, 77, dtype=dtype, seed=9)
    grads = torch.autograd.grad(y, leaves, g)
    pre, tol = oracle.adapter(base, x, a, b, ids, 0.25)[0]
    fn = torch.relu if act == "relu" else torch.sigmoid
    # neither has a slope above 1, so pre's error is not enlarged; __expf
    # and the division are within 8 half steps of 32 bits.  What is rounded
    # to the type is fn(pre), by half a step of fn(pre): near pre = 0 a
    # sigmoid is 1/2, whose half step pre's own does not cover
    _within(y, fn(pre), tol + 8 * oracle.U32
            + fn(pre) * oracle.half_step(dtype) * 1.01)
    out = y.detach()
    slope = (out > 0).float() if act == "relu" else (
        out.float() * (1 - out.float()))
    d = (g.float() * slope).to(dtype)
    _within(grads[0], d.double().cpu(), d.double().cpu().abs() * (
        4 * oracle.U32 + 2 * oracle.half_step(dtype)) + 2.0 ** -24)
    want = oracle.adapter(base, x, a, b, ids, 0.25, grads[0])
    for got, (value, tol) in zip(grads[1:], want[1:]):
        _within(got, value, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "sigmoid"])
@pytest.mark.parametrize("m", [50, 200, 1500])
def test_adapter_act_gradients_in_64_bits(dtype, act, m):
    """Against the gradients of the sum that no one rounded, with the two
    roundings behind an activation in the bound: the slope is taken from the
    rounded output, and its product with g is rounded to the type."""
    base, x, a, b, ids, _ = _adapter_inputs(m, 90, 77, 6, 4, dtype=dtype,
                                            seed=60)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    y = F.adapter_add(*leaves, ids, scale=0.25, act=act)
    g = _randn(m, 77, dtype=dtype, seed=9)
    got = torch.autograd.grad(y, leaves, g)
    (pre, tol), = oracle.adapter(base, x, a, b, ids, 0.25)
    g, half = g.double().cpu(), oracle.half_step(dtype)
    if act == "relu":
        slope = (pre > 0).double()
        off = (pre.abs() <= tol).double()  # either side of 0
    else:
        out = torch.sigmoid(pre)
        slope = out * (1 - out)
        off = tol + 8 * oracle.U32 + out * half * 1.01
        off = off + off * off  # d(y - y^2) <= |dy| + dy^2
    d = g * slope
    err = g.abs() * (off + (slope + off) * (4 * oracle.U32 + half * 1.01))
    if dtype == torch.float16:
        err = err + 2.0 ** -25
    _within(got[0], d, err)
    want = oracle.adapter(base, x, a, b, ids, 0.25, d)
    # what err becomes on its way; 1.01 for its products with the roundings
    # that the oracle's own bounds hold
    chosen = (ids.cpu().unsqueeze(1) == torch.arange(4)).double()
    xa, aa, ba = (t.detach().cpu().double().abs() for t in (x, a, b))
    dz = 0.25 * torch.einsum("me,mn,enr->mr", chosen, err, ba)
    z = 0.25 * torch.einsum("me,mk,erk->mr", chosen, xa, aa)
    more = (torch.einsum("me,mr,erk->mk", chosen, dz, aa),
            torch.einsum("me,mr,mk->erk", chosen, dz, xa),
            torch.einsum("me,mn,mr->enr", chosen, err, z))
    for value, (exact, bound), extra in zip(got[1:], want[1:], more):
        _within(value, exact, bound + extra * 1.01)


@pytest.mark.parametrize("dtype", TYPES)
def test_adapter_layouts(dtype):
    base, x, a, b, ids, scale = _adapter_inputs(48, 65, 33, 5, 3,
                                                dtype=dtype)
    want = F.adapter_add(base, x, a, b, ids, scale=scale)
    wide_x = torch.full((48, 100), math.nan, dtype=dtype, device=DEV)
    wide_x[:, 3:68] = x
    wide_base = torch.full((48, 50), math.nan, dtype=dtype, device=DEV)
    wide_base[:, 1:34] = base
    leaf = wide_x[:, 3:68].detach().requires_grad_()
    got = F.adapter_add(wide_base[:, 1:34], leaf, a, b, ids, scale=scale)
    assert torch.equal(got, want)
    g = _randn(33, 48, dtype=dtype, seed=5).t()  # another order
    (dx,) = torch.autograd.grad(got, leaf, g)
    flat = x.clone().requires_grad_()
    (dw,) = torch.autograd.grad(
        F.adapter_add(base, flat, a, b, ids, scale=scale), flat,
        g.contiguous())
    assert torch.equal(dx, dw)
    other = F.adapter_add(
        base.t().contiguous().t(), x.t().contiguous().t(),
        a.transpose(1, 2).contiguous().transpose(1, 2),
        b.transpose(1, 2).contiguous().transpose(1, 2), ids.int(),
        scale=scale)
    assert torch.equal(other, want)
    shaped = F.adapter_add(base.reshape(4, 12, 33), x.reshape(4, 12, 65), a,
                           b, ids.reshape(4, 12), scale=scale)
    assert torch.equal(shaped.reshape(48, 33), want)
    # one adapter for all, given once and broadcast: its gradient is summed
    one = a[:1].detach().requires_grad_()
    y = F.adapter_add(base, x, one.expand(3, 5, 65), b, ids, scale=scale)
    (da,) = torch.autograd.grad(y, one, g.contiguous())
    each = a[:1].detach().repeat(3, 1, 1).requires_grad_()
    y = F.adapter_add(base, x, each, b, ids, scale=scale)
    (de,) = torch.autograd.grad(y, each, g.contiguous())
    torch.testing.assert_close(da, de.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows_of_any_strides(dtype):
    """Empty batches keep the strides of what they were cut or expanded
    from, also behind contiguous()."""
    base, x, a, b, ids, scale = _adapter_inputs(4, 9, 5, 3, 2, dtype=dtype)
    for cut in (lambda t: t[:0], lambda t: t.t().contiguous().t()[:0],
                lambda t: t[:1, :1].expand(4, t.shape[1])[:0]):
        leaves = [cut(t).detach().requires_grad_() for t in (base, x)]
        leaves += [t.detach().requires_grad_() for t in (a, b)]
        for act in ("none", "relu"):
            y = F.adapter_add(*leaves, ids[:0], scale=scale, act=act)
            assert y.shape == (0, 5)
            grads = torch.autograd.grad(y.sum(), leaves)  # expanded
            assert grads[0].shape == (0, 5) and grads[1].shape == (0, 9)
            assert (grads[2] == 0).all() and (grads[3] == 0).all()
        r = F.token_logprobs(leaves[1], ids[:0], top_k=2)
        assert r.logp.shape == (0,) and r.top_ids.shape == (0, 2)
        (dx,) = torch.autograd.grad(r.logp.sum(), leaves[1])
        assert dx.shape == (0, 9)
        state = F.dropout_state(1, device=DEV)
        y = F.dropout(leaves[1], 0.5, state)
        (dx,) = torch.autograd.grad(y.sum(), leaves[1])
        assert y.shape == dx.shape == (0, 9)


def test_adapter_partial_gradients_and_groups():
    base, x, a, b, ids, scale = _adapter_inputs(90, 40, 30, 4, 3)
    g = _randn(90, 30, seed=6)
    full = [t.detach().requires_grad_() for t in (base, x, a, b)]
    groups = F.adapter_groups(ids, 3)
    y = F.adapter_add(*full, groups, scale=scale)
    every = torch.autograd.grad(y, full, g)
    for i in range(4):
        ts = [t.detach().clone() for t in (base, x, a, b)]
        ts[i].requires_grad_()
        y = F.adapter_add(*ts, ids, scale=scale)
        (one,) = torch.autograd.grad(y, ts[i], g)
        assert torch.equal(one, every[i])


def test_adapter_broken_row_stays_alone():
    base, x, a, b, ids, scale = _adapter_inputs(64, 96, 40, 16, 2)
    ids = torch.arange(64, device=DEV) % 2
    want = F.adapter_add(base, x, a, b, ids, scale=scale)
    x[10, 5] = math.nan
    x[11, 5] = math.inf
    y = F.adapter_add(base, x, a, b, ids, scale=scale)
    ok = torch.ones(64, dtype=torch.bool, device=DEV)
    ok[10:12] = False
    assert torch.equal(y[ok], want[ok])
    assert not torch.isfinite(y[10:12]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_adapter_small_numbers(dtype):
    """Subnormal inputs of the type are not flushed."""
    tiny = torch.finfo(dtype).smallest_normal / 4
    k = 64
    x = torch.full((16, k), tiny, dtype=dtype, device=DEV)
    a = torch.full((1, 4, k), 2.0 ** 13, dtype=dtype, device=DEV)
    b = torch.full((1, 8, 4), 2.0 ** 10, dtype=dtype, device=DEV)
    base = torch.zeros(16, 8, dtype=dtype, device=DEV)
    ids = torch.zeros(16, dtype=torch.int64, device=DEV)
    want = float(x[0, 0]) * k * 2.0 ** 13 * 4 * 2.0 ** 10
    y = F.adapter_add(base, x, a, b, ids)
    assert float(x[0, 0]) > 0 or dtype == torch.float32
    torch.testing.assert_close(y.double(), torch.full_like(y, 1).double()
                               * want, rtol=1e-2, atol=0)


def test_adapter_offsets_past_32_bits():
    m, k, n = 300001, 8192, 24
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(DEV).manual_seed(2))
    base, _, a, b, _, scale = _adapter_inputs(8, k, n, 16, 3,
                                              dtype=torch.bfloat16)
    base = base.repeat(m // 8 + 1, 1)[:m].contiguous()
    ids = torch.arange(m, device=DEV) % 4 - 1
    leaf = x.requires_grad_()
    y = F.adapter_add(base, leaf, a, b, ids, scale=scale)
    g = _randn(8, n, dtype=torch.bfloat16, seed=3).repeat(m // 8 + 1, 1)[:m]
    (dx,) = torch.autograd.grad(y, leaf, g)
    pick = torch.tensor([0, 1, 262144, 262145, 262147, m - 2, m - 1],
                        device=DEV)
    want = oracle.adapter(base[pick], x[pick], a, b, ids[pick], scale,
                          g[pick])
    _within(y[pick], *want[0])
    _within(dx[pick], *want[1])


def test_adapter_captured_and_streams():
    base, x, a, b, ids, scale = _adapter_inputs(
        130, 256, 192, 16, 7, dtype=torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (base, x, a, b)]
    g = _randn(130, 192, dtype=torch.bfloat16, seed=8)
    ids = ids.clone()

    def step():
        y = F.adapter_add(*leaves, ids, scale=scale)
        return (y.detach(),) + torch.autograd.grad(y, leaves, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(on_side, step()):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            leaves[1].copy_(x * (1 + i))
        ids.copy_((ids + 2) % 8 - 1)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, step()):
            assert torch.equal(p, q)


# -- modules and the engine ---------------------------------------------------


@pytest.mark.parametrize("rows", [20, 90, 1500])
def test_operators_together_gpu(rows):
    from tests.test_lm_ops_cpu import check_operators_together

    check_operators_together(DEV, rows)


@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_adapter_linear_rows_of_any_shape(act):
    from sparkflow_amd import nn as snn

    layer = snn.AdapterLinear(12, 7, 3, 4, 0.5, act).to(DEV)
    with torch.no_grad():
        layer.b.normal_()
    x = _randn(2, 5, 12)
    ids = torch.arange(10, device=DEV).reshape(2, 5) % 5 - 1
    flat = x.reshape(10, 12).requires_grad_()
    want = layer(flat, ids.reshape(10))
    (dw,) = torch.autograd.grad(want.sum(), flat)
    # three axes; the same from strided rows
    wide = torch.full((2, 5, 20), math.nan, device=DEV)
    wide[..., 3:15] = x
    for leaf in (x.clone().requires_grad_(),
                 wide[..., 3:15].detach().requires_grad_()):
        for chosen in (ids, F.adapter_groups(ids, 4)):
            got = layer(leaf, chosen)
            assert torch.equal(got, want.reshape(2, 5, 7))
            (dx,) = torch.autograd.grad(got.sum(), leaf)
            assert torch.equal(dx, dw.reshape(2, 5, 12))
    zeros = torch.zeros_like(ids)
    assert torch.equal(layer(x), layer(x, zeros))
    assert torch.equal(layer(x[1, 2]), layer(x, zeros)[1, 2])
    with pytest.raises(RuntimeError, match="shape mismatch"):
        layer(x.reshape(5, 24), ids.reshape(10)[:5])


@pytest.mark.parametrize("act", ["none", "relu"])
def test_layers_on_no_rows(act):
    """An empty batch is an empty answer, and no launch without blocks whose
    error the next operator would report."""
    from sparkflow_amd import nn as snn

    for layer in (snn.AdapterLinear(12, 7, 3, activation=act),
                  snn.AdapterLinear(300, 7, 3, activation=act, bias=False)):
        layer.to(DEV)
        x = torch.empty(0, layer.in_features, device=DEV, requires_grad=True)
        y = layer(x)
        assert y.shape == (0, 7)
        y.sum().backward()
        assert x.grad.shape == x.shape
        assert (layer.a.grad == 0).all() and (layer.b.grad == 0).all()
        assert layer(x.new_empty(3, 0, layer.in_features)).shape == (3, 0, 7)
    w = _randn(6, 4, seed=1)
    x = torch.empty(0, 6, device=DEV, requires_grad=True)
    y = F.linear_act(x, w, None, act)
    assert y.shape == (0, 4)
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert dx.shape == (0, 6)
    assert F.dropout(torch.ones(4, device=DEV), 0.0,
                     F.dropout_state(1, device=DEV)).sum() == 4


@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
def test_frozen_linear_gradient_of_x_gpu(act, monkeypatch):
    """The same with and without frozen weights, and with the activation's
    gradient as a kernel of its own (SPARKFLOW_FUSED_ACTBWD=0)."""
    x, w, b = _randn(33, 20), _randn(20, 17, seed=1), _randn(17, seed=2)
    g = _randn(33, 17, seed=3)

    def dx(weight, bias):
        leaf = x.clone().requires_grad_()
        return torch.autograd.grad(F.linear_act(leaf, weight, bias, act),
                                   leaf, g)[0]

    want = dx(w.clone().requires_grad_(), b)
    assert torch.equal(dx(w, b), want) and torch.equal(dx(w, None),
                                                       dx(w, 0 * b))

    def fused(*args):
        raise AssertionError("the fused kernel was asked for")

    monkeypatch.setenv("SPARKFLOW_FUSED_ACTBWD", "0")
    monkeypatch.setattr(ops.hip, "gemm_dgrad_act", fused, raising=False)
    torch.testing.assert_close(dx(w, b), want)


@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
@pytest.mark.parametrize("fused", ["0", "1"])
def test_trained_layers_on_no_rows(act, fused, monkeypatch):
    """Weights' gradients of an empty batch are zero by every route."""
    monkeypatch.setenv("SPARKFLOW_FUSED_ACTBWD", fused)
    for bias in (True, False):
        x = torch.empty(0, 70, device=DEV, requires_grad=True)
        w = _randn(70, 9, seed=1).requires_grad_()
        b = _randn(9, seed=2).requires_grad_() if bias else None
        leaves = [x, w, b] if bias else [x, w]
        y = F.linear_act(x, w, b, act)
        grads = torch.autograd.grad(y.sum(), leaves)
        assert grads[0].shape == (0, 70)
        assert all((g == 0).all() for g in grads[1:])
        y = F.linear_act(x, w.detach(), None if b is None else b.detach(),
                         act)
        (dx,) = torch.autograd.grad(y.sum(), x)
        assert dx.shape == (0, 70)
        # nothing is left behind, nor on the engine's own thread
        z = torch.ones(4, device=DEV, requires_grad=True)
        assert torch.autograd.grad((z * z).sum(), z)[0].sum() == 8


def test_no_second_derivative():
    """An error, not a silent zero."""
    x = _randn(4, 9).requires_grad_()
    r = F.token_logprobs(x, torch.zeros(4, device=DEV))
    (g,) = torch.autograd.grad(r.logp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        g.sum().backward()
    base, x, a, b, ids, scale = _adapter_inputs(9, 8, 7, 2, 2)
    a.requires_grad_()
    y = F.adapter_add(base, x, a, b, ids, scale=scale)
    (g,) = torch.autograd.grad(y.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        g.sum().backward()


def test_changed_inputs_are_noticed():
    """What backward needs may not change before it runs."""
    state = F.dropout_state(1, device=DEV)
    x = _randn(8).requires_grad_()
    y = F.dropout(x, 0.5, state)
    F.dropout_next(state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    base, x, a, b, ids, scale = _adapter_inputs(9, 8, 7, 2, 2)
    a.requires_grad_()
    y = F.adapter_add(base, x, a, b, ids, scale=scale)
    ids.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    groups = F.adapter_groups(ids, 2)  # keeps its own copy
    want = F.adapter_add(base, x, a, b, groups, scale=scale)
    ids.fill_(1)
    assert torch.equal(F.adapter_add(base, x, a, b, groups, scale=scale),
                       want)


@pytest.mark.parametrize("model", ["dropout", "adapters"])
def test_captured_training_steps(model):
    """The engine's captured step: a new mask at each replay, and weights
    that move."""
    from sparkflow_amd.graph_utils import build_graph
    from sparkflow_amd.parallel.ps import OptimizerSpec, PSCore, TrainConfig
    from sparkflow_amd.parallel.transport import LocalTransport
    from sparkflow_amd.parallel.worker import Worker
    from tests.test_lm_ops_cpu import _adapted_builder, _seeded_dropout_mlp

    width, build = {"dropout": (6, _seeded_dropout_mlp),
                    "adapters": (10, _adapted_builder)}[model]
    graph_json = build_graph(build)
    ps = PSCore(graph_json, OptimizerSpec("adam", 0.01), device=DEV)
    worker = Worker(graph_json, LocalTransport(ps, DEV),
                    TrainConfig(iters=1, seed=0), device=DEV)
    rng = np.random.default_rng(0)
    y = rng.integers(0, 2, (64, 1)).astype(np.float32)
    worker.stage(rng.random((64, width), dtype=np.float32), y)
    worker.run_steps(4, 16, use_graph=True)
    torch.cuda.synchronize()
    drawn = int(worker.module.drop.rng_state[1])
    before = ps.weights.clone()
    seen = []
    for _ in range(3):
        worker.run_steps(2, 16, use_graph=True)
        torch.cuda.synchronize()
        seen.append(ps.weights.clone())
        with torch.no_grad():  # the program's own work between replays
            worker.module(worker.x).sum().item()
    # an eager forward in between draws as well
    assert int(worker.module.drop.rng_state[1]) == drawn + 3 * 3
    for weights in seen:
        assert torch.isfinite(weights).all()
        assert not torch.equal(weights, before)
        before = weights


def test_mnist_cnn_score_gpu():
    from sparkflow_amd.models import mnist_cnn

    model = mnist_cnn().to(DEV)
    x = _randn(6, 784)
    labels = torch.arange(6, device=DEV).float().unsqueeze(1)
    r = model.score(x, labels, top_k=3)
    logp, h, top, ids = oracle.logprobs(model(x), labels.squeeze(1), 3)
    assert torch.equal(r.top_ids.cpu(), ids)
    _within(r.logp, logp, oracle.logprobs_tol(logp, False, 10))
    assert torch.equal(r.top_ids[:, 0].float(), model.predict(x))
