"""What the language-model operators are measured on: dropout whose mask is
never stored, log-probabilities of given tokens, and low-rank adapters of
many requests beside a shared projection.

``run`` computes one pass either in plain torch operations (``own`` false)
or through ``sparkflow_amd.ops.functional`` (``own`` true); ``exact`` gives
the same outputs in 64 bits, written apart from both.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16,
          "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100


def listed():
    return [
        # dropout behind one hidden layer of the MNIST MLP, minibatch 300
        dict(name="dropout_mlp", op="dropout", dtype="fp32", rows=300,
             cols=256, p=0.3, grad=True),
        # a ragged activation: no extent is a multiple of a vector
        dict(name="dropout_odd", op="dropout", dtype="fp16", rows=1023,
             cols=1001, p=0.1, grad=True),
        # the hidden activations of one large training step
        dict(name="dropout_large", op="dropout", dtype="bf16", rows=8192,
             cols=8192, p=0.1, grad=True),
        # this repository's ten-class heads: scores of a minibatch of 300
        dict(name="logprobs_classes", op="logprobs", dtype="fp32", rows=300,
             vocab=10, top=3, masked=False, padded=0.0, grad=True),
        # one decoding step of 16 requests: the chosen tokens' scores and
        # twenty alternatives, some tokens banned
        dict(name="logprobs_decode", op="logprobs", dtype="bf16", rows=16,
             vocab=131072, top=20, masked=True, padded=0.0, grad=False),
        # a fine-tuning step with an entropy term on a padded batch
        dict(name="logprobs_train", op="logprobs", dtype="bf16", rows=4096,
             vocab=32000, top=0, masked=False, padded=0.2, grad=True),
        # rescoring with alternatives in 32 bits, an odd vocabulary
        dict(name="logprobs_rescore", op="logprobs", dtype="fp32", rows=512,
             vocab=50001, top=5, masked=True, padded=0.1, grad=True),
        # one token of each of 32 requests, 64 adapters loaded
        dict(name="adapter_decode", op="adapter", dtype="bf16", rows=32,
             inputs=4096, outputs=4096, rank=16, adapters=64,
             order="shuffled", grad=False),
        # the prompts of many requests, one after another
        dict(name="adapter_prefill", op="adapter", dtype="bf16", rows=8192,
             inputs=4096, outputs=4096, rank=16, adapters=32,
             order="segments", grad=False),
        # adapters beside the first layer of the MNIST MLP, trained
        dict(name="adapter_mlp", op="adapter", dtype="fp32", rows=300,
             inputs=784, outputs=256, rank=8, adapters=4,
             order="shuffled", grad=True),
        # ragged sizes in every extent
        dict(name="adapter_odd", op="adapter", dtype="fp16", rows=777,
             inputs=1000, outputs=513, rank=12, adapters=17,
             order="shuffled", grad=True),
        # a large mixed batch through one wide layer, trained
        dict(name="adapter_train", op="adapter", dtype="bf16", rows=8192,
             inputs=4096, outputs=2048, rank=32, adapters=8,
             order="shuffled", grad=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(
        rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "logprobs", "adapter"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    grad = rng.random() < 0.6
    if op == "dropout":
        rows = _log_int(rng, 1, 8192)
        cols = _log_int(rng, 1, 8192)
        if dtype == "fp32":
            cols = max(1, cols // 2)
        return dict(op=op, dtype=dtype, rows=rows, cols=cols,
                    p=round(rng.uniform(0.02, 0.8), 3), grad=grad)
    if op == "logprobs":
        vocab = _log_int(rng, 2, 262144)
        most = (1 << 27) // vocab // (2 if dtype == "fp32" else 1)
        rows = _log_int(rng, 1, max(1, min(8192, most)))
        top = min(vocab, rng.choice([0, 0, 1, 5, 20, 32]))
        while rows * vocab * max(1, top) > 1 << 28:
            rows = max(1, rows // 2)
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=top,
                    masked=vocab > 64 and rng.random() < 0.5,
                    padded=rng.choice([0.0, 0.1, 0.3]), grad=grad)
    inputs = _log_int(rng, 16, 4096)
    outputs = _log_int(rng, 16, 4096)
    rank = _log_int(rng, 1, 64)
    adapters = _log_int(rng, 1, 64)
    rows = _log_int(rng, 1, 8192)
    while rows * (inputs + outputs) * rank * adapters > 1 << 34:
        rows = max(1, rows // 2)
    return dict(op=op, dtype=dtype, rows=rows, inputs=inputs,
                outputs=outputs, rank=rank, adapters=adapters,
                order=rng.choice(["segments", "shuffled"]), grad=grad)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda",
                            dtype=torch.float32) * std).to(dtype)

    def whole(hi, *shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda")

    s = {"case": case}
    m = case["rows"]
    if case["op"] == "dropout":
        s["x"] = normal(m, case["cols"])
        s["state"] = whole(1 << 62, 2)  # the generator's key and offset
        if case["grad"]:
            s["g"] = normal(m, case["cols"])
    elif case["op"] == "logprobs":
        v = case["vocab"]
        s["logits"] = normal(m, v, std=3.0)
        s["tokens"] = whole(v, m)
        if case["masked"]:
            # banned tokens, never the one that is scored
            ban = torch.rand(m, v, generator=gen, device="cuda") < 0.05
            ban.scatter_(1, s["tokens"].unsqueeze(1), False)
            s["logits"].masked_fill_(ban, -math.inf)
        if case["padded"]:
            pad = torch.rand(m, generator=gen, device="cuda")
            s["tokens"].masked_fill_(pad < case["padded"], IGNORE)
        if case["grad"]:
            s["g_logp"] = normal(m, std=1.0 / m, dtype=torch.float32)
            s["g_entropy"] = normal(m, std=0.1 / m, dtype=torch.float32)
            s["g_top"] = normal(m, case["top"], std=0.1 / m,
                                dtype=torch.float32)
    else:
        k, n = case["inputs"], case["outputs"]
        r, e = case["rank"], case["adapters"]
        s["x"] = normal(m, k)
        s["base"] = normal(m, n)  # what the shared projection gave
        s["a"] = normal(e, r, k, std=k ** -0.5)
        s["b"] = normal(e, n, r, std=r ** -0.5)
        s["scale"] = torch.rand(e, generator=gen, device="cuda") + 0.5
        ids = whole(e + 1, m) - 1  # -1: a request without an adapter
        if case["order"] == "segments":
            ids = ids[torch.sort(whole(max(1, m // 256), m))[0]]
        s["ids"] = ids
        if case["grad"]:
            s["g"] = normal(m, n)
    if case["grad"]:
        for name in ("x", "logits", "base", "a", "b"):
            if name in s:
                s[name].requires_grad_()
    return s


# -- the framework's operators ------------------------------------------------


def _own(s):
    from sparkflow_amd.ops import functional as F

    case = s["case"]
    if case["op"] == "dropout":
        y = F.dropout(s["x"], case["p"], s["state"])
        if not case["grad"]:
            return {"y": y}
        return {"y": y.detach(),
                "dx": torch.autograd.grad(y, s["x"], s["g"])[0]}
    if case["op"] == "logprobs":
        r = F.token_logprobs(s["logits"], s["tokens"], top_k=case["top"],
                             ignore_index=IGNORE)
        out = {"logp": r.logp, "entropy": r.entropy, "top": r.top_logp,
               "ids": r.top_ids}
        if case["grad"]:
            out = {name: t.detach() for name, t in out.items()}
            roots, gs = [r.logp, r.entropy], [s["g_logp"], s["g_entropy"]]
            if case["top"]:
                roots, gs = roots + [r.top_logp], gs + [s["g_top"]]
            out["dlogits"] = torch.autograd.grad(roots, s["logits"], gs)[0]
        return out
    y = F.adapter_add(s["base"], s["x"], s["a"], s["b"], s["ids"],
                      scale=s["scale"])
    if not case["grad"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [s["base"], s["x"], s["a"], s["b"]],
                                s["g"])
    return dict(zip(("y", "dbase", "dx", "da", "db"), (y.detach(),) + grads))


# -- plain forms --------------------------------------------------------------


def _mul32(a, c):
    """High and low 32 bits of a * c, for 32-bit values held in int64."""
    high = (a * (c >> 16) + ((a * (c & 0xFFFF)) >> 16)) >> 16
    return high, (a * c) & 0xFFFFFFFF


def _random_words(state, n):
    """n words of Philox4x32 with 10 rounds (Salmon et al. 2011, "Parallel
    random numbers: as easy as 1, 2, 3"), four to a counter; the counter is
    (element // 4, offset) and the key is the seed, 64 bits each."""
    at = torch.arange((n + 3) // 4, device=state.device)
    key, offset = state[0], state[1]
    c0, c1 = at & 0xFFFFFFFF, at >> 32
    c2 = (offset & 0xFFFFFFFF).expand_as(at)
    c3 = ((offset >> 32) & 0xFFFFFFFF).expand_as(at)
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mul32(0xD2511F53, c0)
        h1, l1 = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0 = (k0 + 0x9E3779B9) & 0xFFFFFFFF
        k1 = (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _plain_dropout(s):
    x, keep = s["x"].detach(), 1.0 - s["case"]["p"]
    words = _random_words(s["state"], x.numel()).reshape(x.shape)
    kept = words < round(keep * 2 ** 32)

    def drop(t):
        return torch.where(kept, t.float() * (1.0 / keep), 0.0).to(t.dtype)

    out = {"y": drop(x)}
    if s["case"]["grad"]:
        out["dx"] = drop(s["g"])
    return out


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].detach().float()
    m, v = x.shape
    live = s["tokens"] != IGNORE
    token = torch.where(live, s["tokens"], 0).unsqueeze(1)
    shift = x.amax(1, keepdim=True)
    lse = (x - shift).exp().sum(1, keepdim=True).log() + shift
    logp = x - lse
    prob = logp.exp()
    entropy = -torch.where(prob > 0, prob * logp, 0.0).sum(1)
    # the largest first, equal ones by the lowest id: a value's bits in an
    # order that integers keep, the id behind them
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
    order = order + torch.arange(v - 1, -1, -1, device=x.device)
    ids = v - 1 - (order.topk(case["top"], 1).values & 0xFFFFFFFF)
    gone = ~live.unsqueeze(1)
    out = {"logp": torch.where(live, logp.gather(1, token)[:, 0], 0.0),
           "entropy": torch.where(live, entropy, 0.0),
           "top": torch.where(gone, 0.0, logp.gather(1, ids)),
           "ids": torch.where(gone, -1, ids)}
    if case["grad"]:
        g, h, t = s["g_logp"], s["g_entropy"], s["g_top"]
        d = torch.where(prob > 0, prob * (logp + entropy.unsqueeze(1)), 0.0)
        d = -h.unsqueeze(1) * d - (g + t.sum(1)).unsqueeze(1) * prob
        d = d.scatter_add(1, token, g.unsqueeze(1)).scatter_add(1, ids, t)
        d = torch.where(gone, 0.0, d)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_adapter(s):
    x, base = s["x"].detach(), s["base"].detach()
    a, b = s["a"].detach().float(), s["b"].detach().float()
    e, r, k = a.shape
    n, m = b.shape[1], x.shape[0]
    # every row through all adapters side by side, the others' shares
    # taken out between the two products
    mine = s["ids"].unsqueeze(1) == torch.arange(e, device=x.device)
    mine = (mine.float() * s["scale"]).repeat_interleave(r, 1)
    down = a.reshape(e * r, k)
    up = b.transpose(1, 2).reshape(e * r, n)
    z = (x.float() @ down.t()) * mine
    out = {"y": (base.float() + z @ up).to(base.dtype)}
    if s["case"]["grad"]:
        g = s["g"].float()
        dz = (g @ up.t()) * mine
        db = (z.t() @ g).reshape(e, r, n).transpose(1, 2)
        out["dbase"] = s["g"].to(base.dtype)
        out["dx"] = (dz @ down).to(x.dtype)
        out["da"] = (dz.t() @ x.float()).reshape(e, r, k).to(x.dtype)
        out["db"] = db.contiguous().to(x.dtype)
    return out


_PLAIN = {"dropout": _plain_dropout, "logprobs": _plain_logprobs,
          "adapter": _plain_adapter}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def work(case):
    m, size = case["rows"], SIZE[case["dtype"]]
    passes = 2 if case["grad"] else 1
    if case["op"] == "dropout":
        n = m * case["cols"]
        return {"bytes": 2 * n * size * passes + 16, "flops": n * passes}
    if case["op"] == "logprobs":
        n = m * case["vocab"]
        rows = m * (16 + 12 * case["top"]) * passes
        return {"bytes": n * size * passes + rows,
                "flops": n * (5 if case["grad"] else 3)}
    k, n, r = case["inputs"], case["outputs"], case["rank"]
    weights = min(m, case["adapters"]) * r * (k + n) * size
    flops = 2 * m * r * (k + n)
    if not case["grad"]:
        return {"bytes": m * (k + 2 * n) * size + weights + 8 * m,
                "flops": flops}
    return {"bytes": m * (2 * k + 4 * n) * size + 2 * weights + 8 * m,
            "flops": 3 * flops}


# -- the same outputs from the definitions, in 64 bits ------------------------


def _exact_words(seed, offset, n):
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    words = np.empty(((n + 3) // 4, 4), dtype=np.uint32)
    step = 1 << 18
    for start in range(0, len(words), step):
        at = np.arange(start, min(len(words), start + step), dtype=u64)
        ctr = [at & low, at >> u64(32), np.full_like(at, offset & 0xFFFFFFFF),
               np.full_like(at, offset >> 32)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            even, odd = ctr[0] * u64(0xD2511F53), ctr[2] * u64(0xCD9E8D57)
            ctr = [(odd >> u64(32)) ^ ctr[1] ^ u64(key[0]), odd & low,
                   (even >> u64(32)) ^ ctr[3] ^ u64(key[1]), even & low]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32,
                   (key[1] + 0xBB67AE85) % 2 ** 32]
        words[start:start + step] = np.stack(ctr, 1)
    return words.reshape(-1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "dropout":
            key, offset = (int(v) % 2 ** 64 for v in s["state"].cpu())
            words = _exact_words(key, offset, s["x"].numel())
            kept = words < round((1.0 - case["p"]) * 2 ** 32)
            kept = torch.from_numpy(kept).cuda().reshape(s["x"].shape)
            out = {"y": s["x"].double() * kept / (1.0 - case["p"])}
            if case["grad"]:
                out["dx"] = s["g"].double() * kept / (1.0 - case["p"])
            return out
        if case["op"] == "logprobs":
            return _exact_logprobs(s)
        return _exact_adapter(s)


def _exact_logprobs(s):
    case = s["case"]
    live = (s["tokens"] != IGNORE).double()
    logp = torch.log_softmax(s["logits"].double(), 1)
    p = torch.exp(logp)
    finite = torch.where(p == 0, torch.zeros_like(logp), logp)
    entropy = -(p * finite).sum(1)
    token = s["tokens"].clamp(min=0)
    rank = torch.sort(s["logits"].double(), dim=1, descending=True,
                      stable=True)
    ids = rank.indices[:, :case["top"]]
    rows = torch.arange(len(token), device=token.device)
    # the score of a padded row is zero; its alternatives are unnamed
    out = {"logp": finite[rows, token] * live, "entropy": entropy * live,
           "top": None, "ids": None}
    if case["top"]:
        top = torch.gather(logp, 1, ids)
        out["top"] = torch.where(live[:, None] > 0, top, 0 * live[:, None])
    if case["grad"]:
        hot = torch.zeros_like(p)
        hot[rows, token] += s["g_logp"].double()
        for j in range(case["top"]):
            hot[rows, ids[:, j]] += s["g_top"][:, j].double()
        share = hot.sum(1, keepdim=True)
        d = hot - p * share
        d -= s["g_entropy"].double()[:, None] * p * (
            finite + entropy[:, None])
        out["dlogits"] = d * live[:, None]
    return out


def _exact_adapter(s):
    case = s["case"]
    x, a, b = s["x"].double(), s["a"].double(), s["b"].double()
    y = s["base"].double().clone()
    g = s["g"].double() if case["grad"] else None
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(case["adapters"]):
        at = (s["ids"] == i).nonzero()[:, 0]
        scale = float(s["scale"][i])
        down = x[at] @ a[i].T
        y[at] += scale * (down @ b[i].T)
        if case["grad"]:
            back = scale * (g[at] @ b[i])
            dx[at] = back @ a[i]
            da[i] = back.T @ x[at]
            db[i] = scale * (g[at].T @ down)
    if not case["grad"]:
        return {"y": y}
    return {"y": y, "dbase": g, "dx": dx, "da": da, "db": db}
