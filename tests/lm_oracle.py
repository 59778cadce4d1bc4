"""64-bit definitions of the language-model operators, and how far a
kernel that sums in 32 bits may be from them.

A rounding to type T is off by at most half a step, ``finfo(T).eps / 2`` of
the value (fp32 2^-24).
"""
import math

import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# -- dropout ------------------------------------------------------------------


def philox_words(seed, offset, first_block, blocks):
    """Philox4x32-10 (Salmon et al. 2011) at the counters (block, offset)
    under the key seed, in Python's own whole numbers where it is short and
    numpy's 64 bits where it runs over the blocks."""
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    at = np.arange(first_block, first_block + blocks, dtype=u64)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    c = [at & low, at >> u64(32), np.full_like(at, offset % 2 ** 32),
         np.full_like(at, offset // 2 ** 32)]
    k = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        p, q = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(q >> u64(32)) ^ c[1] ^ u64(k[0]), q & low,
             (p >> u64(32)) ^ c[3] ^ u64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, 1).reshape(-1).astype(np.int64)


def kept(state, p, n, first=0):
    """Which of the elements first .. first + n - 1 stay (first % 4 == 0)."""
    seed, offset = (int(v) for v in state.cpu())
    words = philox_words(seed, offset, first // 4, (n + 3) // 4)[:n]
    return torch.from_numpy(words < round((1.0 - p) * 2 ** 32))


def dropout(x, state, p):
    keep = kept(state, p, x.numel()).reshape(x.shape)
    y = x.cpu().double() / (1.0 - p) if p < 1 else x.cpu().double()
    return torch.where(keep, y, torch.zeros_like(y))


# -- log-probabilities --------------------------------------------------------


def logprobs(logits, tokens, k, ignore=-100):
    """(logp, entropy, top, ids) row by row, on finite and -inf logits."""
    x = logits.detach().cpu().double()
    tokens = tokens.cpu().long()
    m, c = x.shape
    out = [torch.zeros(m, dtype=torch.float64) for _ in range(2)]
    out += [torch.zeros(m, k, dtype=torch.float64),
            torch.full((m, k), -1, dtype=torch.int64)]
    for i in range(m):
        if int(tokens[i]) == ignore:
            continue
        row = x[i]
        if torch.isneginf(row).all():
            logp = row
            h = 0.0
        else:
            best = row.max()
            logp = row - best - torch.log(torch.exp(row - best).sum())
            p = torch.exp(logp)
            h = float(-(p[p > 0] * logp[p > 0]).sum())
        t = int(tokens[i])
        out[0][i] = logp[t] if 0 <= t < c else math.nan
        out[1][i] = h
        ids = torch.from_numpy(
            np.lexsort((np.arange(c), -row.numpy()))[:k].copy())
        out[2][i] = logp[ids]
        out[3][i] = ids
    return out


def logprobs_grad(logits, tokens, k, gs, ignore=-100):
    """dlogits by the formula, and how far 32-bit sums may be from it."""
    x = logits.detach().cpu().double()
    tokens = tokens.cpu().long()
    m, c = x.shape
    _, h, _, ids = logprobs(logits, tokens, k, ignore)
    zero = torch.zeros(m, dtype=torch.float64)
    g, gh = (zero if t is None else t.cpu().double() for t in gs[:2])
    gt = torch.zeros(m, k, dtype=torch.float64) if gs[2] is None \
        else gs[2].cpu().double()
    dx, tol = torch.zeros_like(x), torch.zeros_like(x)
    n = sum_error(c)
    for i in range(m):
        if int(tokens[i]) == ignore or torch.isneginf(x[i]).all():
            continue
        logp = torch.log_softmax(x[i], 0)
        p = torch.exp(logp)
        logp = torch.where(p == 0, torch.zeros_like(p), logp)
        hot = torch.zeros(c, dtype=torch.float64)
        hot[tokens[i]] += g[i]
        hot.index_add_(0, ids[i], gt[i])
        share = float(g[i] + gt[i].sum())
        dx[i] = hot - p * (share + gh[i] * (logp + h[i]))
        size = abs(g[i]) + gt[i].abs().sum() + gh[i].abs() * (
            logp.abs() + h[i] + 1)
        # e^(x - lse): the exponent's rounding and lse's own error; the
        # entropy's error; one rounding for each product and sum
        tol[i] = p * size * (2 * logp.abs() + 2 * n + k + 16) * U32
        tol[i] += hot.abs() * 4 * U32
    tol += dx.abs() * half_step(logits.dtype) + 1e-37
    if logits.dtype == torch.float16:
        tol += 2.0 ** -25  # half a step of its subnormal numbers
    return dx, tol


def sum_error(c):
    """Half steps that log(sum of c exponentials) may be off.  A term
    e^d is off by |d| log2(e) + 4 (the product and the exponential), which
    weighted by the terms is at most 1.45 log c; the sum by one step an
    addition: c / 64 in a thread at most, its rescalings (one a vector at
    most, two roundings each), and 12 where threads join."""
    return 1.45 * math.log(c + 1) + 4 + 3 * (c / 64 + 1) + 12


def logprobs_tol(want, entropy, c):
    """For values whose size is |want|: the logarithm, the difference and
    the rounding behind the sum's error."""
    size = torch.where(torch.isfinite(want), want.abs(),
                       torch.zeros_like(want))
    n = sum_error(c) * (1 + (math.log(c + 1) if entropy else 0))
    return (2 * n + 8 + 8 * size + 2 * math.log(c + 1)) * U32


# -- low-rank adapters --------------------------------------------------------


def depth(n):
    """Additions that one of n terms goes through at most: sums are split
    over four waves at least, and 40 covers the steps that join them."""
    return n / 4 + 40


def adapter(base, x, a, b, ids, scale, g=None):
    """y (and dx, da, db for the gradient g of y) by adapter in 64 bits,
    each with the bound of a computation that sums in 32 bits and rounds
    once to the inputs' type."""
    dtype = x.dtype
    base, x, a, b = (t.detach().cpu().double() for t in (base, x, a, b))
    ids = ids.cpu()
    e, r, k = a.shape
    n, m = b.shape[1], x.shape[0]
    y, dx = base.clone(), torch.zeros_like(x)
    ty, tx = base.abs() * 2 * U32, torch.zeros_like(x)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    ta, tb = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(e):
        at = (ids == i).nonzero().squeeze(1)
        if not len(at):
            continue
        s = float(scale[i]) if isinstance(scale, torch.Tensor) else scale
        s_err = 2 * U32  # the scale in 32 bits, and its product
        xa, ba = x[at], b[i].abs()
        z = s * (xa @ a[i].T)
        z_size = abs(s) * (xa.abs() @ a[i].abs().T)
        z_err = z_size * (depth(k) * U32 + s_err)
        y[at] += z @ b[i].T
        ty[at] += z_err @ ba.T + (z.abs() + z_err) @ ba.T * (r + 4) * U32
        if g is None:
            continue
        ga = g[at].detach().cpu().double()
        dz = s * (ga @ b[i])
        dz_err = abs(s) * (ga.abs() @ ba) * (depth(n) * U32 + s_err)
        dx[at] = dz @ a[i]
        tx[at] = dz_err @ a[i].abs() + (
            (dz.abs() + dz_err) @ a[i].abs()) * (r + 4) * U32
        da[i], db[i] = dz.T @ xa, ga.T @ z
        d = depth(len(at)) * U32
        ta[i] = dz_err.T @ xa.abs() + (dz.abs() + dz_err).T @ xa.abs() * d
        tb[i] = ga.abs().T @ z_err + ga.abs().T @ (z.abs() + z_err) * d

    def rounded(t, tol):
        tol = tol + (t.abs() + tol) * half_step(dtype) + 1e-37
        return tol + (2.0 ** -25 if dtype == torch.float16 else 0)

    out = [(y, rounded(y, ty))]
    if g is not None:
        out += [(dx, rounded(dx, tx)), (da, rounded(da, ta)),
                (db, rounded(db, tb))]
    return out
