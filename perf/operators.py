"""Top alternatives, log-probabilities of given tokens and the router's balance loss: what is measured of them.

Each case is one pass through one operator as a user's program calls it: a scorer that wants a response's
log-probabilities with the best alternatives of every position, a student that needs its log-probabilities of the
tokens that a teacher stored, forward and backward, each of them from materialised logits and from the final hidden
states through the head, and the balance loss of a mixture of experts, forward and backward, beside the step's loss.

``run`` computes the operators in plain torch operations in 32 bits where ``own`` is false, and calls the package
where it is true.  ``exact`` states the same definitions in 64 bits.  All inputs are synthetic and made on the GPU from
the seed.

Definitions.  ``z``: a row's logits (through the head: ``cap * tanh(hidden . weight / cap) / temperature``).
``lse = log sum exp z``; a token's log-probability is ``z[token] - lse``, 0 for an id outside the vocabulary; the
entropy is ``lse - sum softmax(z) z``.  The top alternatives are the k largest logits in descending order, equal ones by
ascending id.  For a router's scores ``p`` (softmax of a token's logits, or their sigmoids divided by their sum), its k
largest logits chosen per token (or the experts that are given), over the T unmasked tokens of a batch or of a
sequence:  ``sum_e E / (k T) c_e * (sum_t p_te) / T`` with the choices ``c_e`` counted as constants; the mean over
the sequences that have tokens and over the layers.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # set by the program that imports this file

# hidden, vocabulary: head shapes of the benchmark, then generic ones
HEADS = ((896, 151936), (2880, 201088), (4096, 151936), (2048, 32768), (1024, 50257))
VOCABS = (151936, 201088, 32768, 50257)
EXPERTS = ((8, 2), (32, 4), (60, 4), (64, 6), (128, 8), (160, 6), (256, 8), (512, 10))

MAX_FLOPS = 2.0 * 8192 * 4096 * 151936
MAX_LOGITS = 4096 * 151936
MAX_ROUTER = 48 * 8192 * 128


def listed():
    return [
        # A decoder that reports the best alternatives of the one token that it is about to sample.
        dict(name="top_one_token", kind="top", tokens=1, vocab=151936, k=20, bits=16, labels=False, banned=0, grad=False),
        # A decode batch under a constraint that bans part of the vocabulary: fp32 logits, an odd number of rows.
        dict(name="top_decode_batch", kind="top", tokens=61, vocab=201088, k=5, bits=32, labels=True, banned=1000,
             grad=False),
        # Scoring a micro-batch whose logits are there: log-probabilities, entropy and twenty alternatives.
        dict(name="top_scoring", kind="top", tokens=4096, vocab=151936, k=20, bits=16, labels=True, banned=0, grad=False),
        # The same as part of a loss, on an odd vocabulary whose rows start off every boundary: with the gradient.
        dict(name="top_odd_vocab_grad", kind="top", tokens=2047, vocab=50257, k=64, bits=16, labels=True, banned=0,
             grad=True),
        # A student on a short response: log-probabilities of a teacher's stored alternatives, with the gradient.
        dict(name="tokens_short_grad", kind="tokens", tokens=187, vocab=151936, k=8, bits=16),
        # The same over a micro-batch, more alternatives, fp32 logits.
        dict(name="tokens_micro_batch_grad", kind="tokens", tokens=1500, vocab=151936, k=32, bits=32),
        # A decode step from the hidden states on: alternatives of a few tokens through the small head.
        dict(name="head_top_decode", kind="head_top", tokens=8, hidden=896, vocab=151936, k=20, temperature=1.0,
             softcap=0.0),
        # A teacher scoring a whole micro-batch through the large head, whose logits do not fit anywhere.
        dict(name="head_top_scoring", kind="head_top", tokens=8192, hidden=4096, vocab=151936, k=20, temperature=1.0,
             softcap=0.0),
        # A student's step on a ragged micro-batch of the small head: sixty-four stored alternatives, with gradients.
        dict(name="head_tokens_grad", kind="head_tokens", tokens=1001, hidden=896, vocab=151936, k=64, temperature=1.0,
             softcap=0.0),
        # The same on the large vocabulary.
        dict(name="head_tokens_large_grad", kind="head_tokens", tokens=2500, hidden=2880, vocab=201088, k=16,
             temperature=1.0, softcap=0.0),
        # One layer's router on a short packed batch, balanced sequence by sequence: latency.
        dict(name="balance_sequences_short", kind="balance", layers=1, tokens=1021, experts=60, k=4, bits=32,
             score="sigmoid", given=False, sequences=True, mask_bits=64),
        # All layers' routers of a micro-batch at once, choices counted from the logits.
        dict(name="balance_layers", kind="balance", layers=48, tokens=8192, experts=128, k=8, bits=16, score="softmax",
             given=False, sequences=False, mask_bits=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; token counts are spread over their logarithm."""
    kind = rng.choice(("top", "top", "top", "tokens", "tokens", "head_top", "head_top", "head_tokens", "balance",
                       "balance", "balance"))
    if kind in ("top", "tokens"):
        vocab = rng.choice(VOCABS + (_log_int(rng, 1000, 260000),))
        bits = rng.choice((16, 16, 32))
        grad = kind == "tokens" or rng.random() < 0.4
        cost = bits // 16 * (2 if grad else 1)
        tokens = _log_int(rng, 1, max(2, min(8192, MAX_LOGITS // (vocab * cost))))
        if kind == "tokens":
            return dict(kind=kind, tokens=tokens, vocab=vocab, k=_log_int(rng, 1, 128), bits=bits)
        return dict(kind=kind, tokens=tokens, vocab=vocab, k=_log_int(rng, 1, 128), bits=bits,
                    labels=rng.random() < 0.7, banned=rng.choice((0, 0, 333)), grad=grad)
    if kind in ("head_top", "head_tokens"):
        hidden, vocab = rng.choice(HEADS)
        per_token = (2.0 if kind == "head_top" else 6.0) * hidden * vocab
        tokens = min(_log_int(rng, 1, 8192), int(0.9 * MAX_FLOPS / per_token))
        return dict(kind=kind, tokens=tokens, hidden=hidden, vocab=vocab, k=_log_int(rng, 1, 64),
                    temperature=rng.choice((1.0, 1.0, 0.7)),
                    softcap=rng.choice((0.0, 0.0, 30.0)))
    experts, k = rng.choice(EXPERTS)
    bits, layers = rng.choice((16, 32)), rng.choice((1, 4, 24, 48))
    tokens = _log_int(rng, 1, max(2, min(16384, MAX_ROUTER // (experts * layers * (bits // 16)))))
    return dict(kind="balance", layers=layers, tokens=tokens, experts=experts, k=k, bits=bits,
                score=rng.choice(("softmax", "sigmoid")), given=rng.random() < 0.4, sequences=rng.random() < 0.5,
                mask_bits=rng.choice((0, 32, 64)))


# --------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ids(g, vocab, *shape):
    return torch.randint(0, vocab, shape, generator=g, device="cuda")


def _alternatives(g, vocab, n, k):
    """Ids that another model stored per position: distinct within a row up to chance, one in fifty a filler (-1)."""
    ids = _ids(g, vocab, n, k)
    return torch.where(torch.rand(n, k, generator=g, device="cuda") < 0.02, torch.full_like(ids, -1), ids)


def _upstream(g, n, *tail):
    """Gradients of a token-mean loss on log-probabilities, and a small pull on the entropy."""
    return _randn(g, n, *tail) / n, -0.01 / n + 0.001 * _randn(g, n) / n


def _prepare_logits(c, g):
    n, v = c["tokens"], c["vocab"]
    k = min(c["k"], v)
    z = torch.empty(n, v, device="cuda").normal_(0.0, 2.0, generator=g)
    at = _ids(g, v, n)
    z[torch.arange(n, device="cuda"), at] += 9.0  # a trained model is sure of most tokens
    z = z.to(torch.bfloat16 if c["bits"] == 16 else torch.float32)
    s = dict(c, k=k, logits=z)
    if c["kind"] == "tokens":
        ids = _alternatives(g, v, n, k)
        ids[:, 0] = at
        s.update(ids=ids)
        s["g_ids"], s["g_en"] = _upstream(g, n, k)
        z.requires_grad_(True)
        return s
    if c["banned"]:  # a constraint on what may be sampled
        z[:, _ids(g, v, c["banned"])] = -math.inf
        z[:, v // 2] = 0.5
    s["labels"] = torch.where(z[torch.arange(n, device="cuda"), at] > -math.inf, at, v // 2) if c["labels"] else None
    if c["grad"]:
        s["g_top"], s["g_en"] = _upstream(g, n, k)
        s["g_lp"] = _randn(g, n) / n
        z.requires_grad_(True)
    return s


def _head_operands(c, g, gridded):
    """Hidden states and head weight in bf16, logits of a standard deviation of about 2.  ``gridded``: on a grid so
    coarse that every sum of their products is exact in 32 bits whatever its order, so that equal logits are equal
    for every implementation and the ids of the largest are defined."""
    n, h, v = c["tokens"], c["hidden"], c["vocab"]
    shift = 2.0 ** -round(math.log2(math.sqrt(h)) - 1.0)
    w = _randn(g, v, h)
    if gridded:
        w = (w * 4.0).round_().clamp_(-12, 12).div_(4.0)
    at = _ids(g, v, n)
    hid = _randn(g, n, h) + 0.08 * w[at]  # a trained head: the token that follows stands out
    if gridded:
        hid = (hid * 32.0).round_().clamp_(-128, 128).div_(32.0)
    return hid.to(torch.bfloat16), w.mul_(shift).to(torch.bfloat16), at


def _prepare_head(c, g):
    n, v = c["tokens"], c["vocab"]
    top = c["kind"] == "head_top"
    hid, w, at = _head_operands(c, g, top)
    s = dict(c, h=hid, w=w)
    if top:
        s["labels"] = at
        return s
    ids = _alternatives(g, v, n, c["k"])
    ids[:, 0] = at
    s.update(ids=ids)
    s["g_ids"], s["g_en"] = _upstream(g, n, c["k"])
    hid.requires_grad_(True)
    w.requires_grad_(True)
    return s


def _offsets(total, r):
    lens, left = [], total
    while left > 0:
        x = min(max(int(round(math.exp(r.gauss(5.5, 0.8)))), 1), left)
        lens.append(x)
        left -= x
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _prepare_balance(c, g, r):
    n, e, k = c["tokens"], c["experts"], c["k"]
    dtype = torch.bfloat16 if c["bits"] == 16 else torch.float32
    logits = [(1.5 * _randn(g, n, e) + _randn(g, e)).to(dtype).requires_grad_(True) for _ in range(c["layers"])]
    s = dict(c, logits=logits, ids=None, mask=None, cu=None)
    if c["given"]:  # a router that chose by other scores than these logits
        s["ids"] = [torch.rand(n, e, generator=g, device="cuda").argsort(1)[:, :k].contiguous() for _ in logits]
    if c["mask_bits"]:
        m = torch.rand(n, generator=g, device="cuda") < 0.7
        m[0] = True
        s["mask"] = m.to(torch.int64) if c["mask_bits"] == 64 else m.to(torch.float32)
    if c["sequences"]:
        s["cu"] = _offsets(n, r)
    s["g_loss"] = torch.full((), 0.01, device="cuda")  # the loss's coefficient
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "balance":
        return _prepare_balance(case, g, random.Random(seed))
    return (_prepare_logits if case["kind"] in ("top", "tokens") else _prepare_head)(case, g)


# --------------------------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# --------------------------------------------------------------------------------------------------------------

def _largest(z, k):
    """Ids of each row's k largest values, descending, equal ones by ascending id."""
    out = []
    v = z.shape[1]
    below = torch.arange(v - 1, -1, -1, device=z.device)
    for rows in z.split(max(1, (1 << 27) // v)):
        bits = (rows + 0.0).contiguous().view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)  # integers in the order of the values
        out.append(v - 1 - (((order << 32) | below).topk(k, dim=1).values & 0xFFFFFFFF))
    return torch.cat(out)


def _statistics(z):
    m = z.max(1, keepdim=True).values
    ex = torch.exp(z - m)
    total = ex.sum(1, keepdim=True)
    lse = m + torch.log(total)
    p = ex / total
    entropy = (lse - (p * torch.where(p > 0, z, torch.zeros_like(z))).sum(1, keepdim=True)).squeeze(1)
    return lse, p, entropy


def _pick(z, lse, ids):
    ok = (ids >= 0) & (ids < z.shape[1])
    return torch.where(ok, z.gather(1, torch.where(ok, ids, torch.zeros_like(ids))) - lse, torch.zeros_like(lse))


def _dlogits(z, lse, p, entropy, ids, g_ids, g_entropy):
    """Gradient of sum g_ids * logprob[ids] + sum g_entropy * entropy with respect to z."""
    ok = (ids >= 0) & (ids < z.shape[1])
    g = torch.where(ok, g_ids, torch.zeros_like(g_ids))
    log_p = torch.where(p > 0, z - lse, torch.zeros_like(z))
    d = -p * (g.sum(1, keepdim=True) + g_entropy[:, None] * (log_p + entropy[:, None]))
    return d.scatter_add_(1, torch.where(ok, ids, torch.zeros_like(ids)), g)


def _plain_top(s):
    z = s["logits"].detach().float()
    lse, p, entropy = _statistics(z)
    ids = _largest(z, s["k"])
    out = [entropy, z.gather(1, ids) - lse, ids]
    if s["labels"] is not None:
        out.append(_pick(z, lse, s["labels"][:, None]).squeeze(1))
    if s["grad"]:
        at, g = ids, s["g_top"]
        if s["labels"] is not None:
            at, g = torch.cat([s["labels"][:, None], ids], 1), torch.cat([s["g_lp"][:, None], g], 1)
        out.append(_dlogits(z, lse, p, entropy, at, g, s["g_en"]).to(s["logits"].dtype))
    return out


def _plain_tokens(s):
    z = s["logits"].detach().float()
    lse, p, entropy = _statistics(z)
    grad = _dlogits(z, lse, p, entropy, s["ids"], s["g_ids"], s["g_en"]).to(s["logits"].dtype)
    return [_pick(z, lse, s["ids"]), entropy, grad]


def _head_logits(s):
    raw = s["h"].detach().float() @ s["w"].detach().float().t()
    z = raw
    if s["softcap"]:
        z = s["softcap"] * torch.tanh(raw / s["softcap"])
    return raw, z / s["temperature"]


def _plain_head_top(s):
    raw, z = _head_logits(s)
    lse, _, entropy = _statistics(z)
    ids = _largest(raw, s["k"])  # the cap and the temperature keep the order of what they do not make equal
    return [entropy, z.gather(1, ids) - lse, ids, _pick(z, lse, s["labels"][:, None]).squeeze(1)]


def _plain_head_tokens(s):
    _, z = _head_logits(s)
    lse, p, entropy = _statistics(z)
    d = _dlogits(z, lse, p, entropy, s["ids"], s["g_ids"], s["g_en"]) / s["temperature"]
    if s["softcap"]:
        d = d * (1.0 - (z * (s["temperature"] / s["softcap"])) ** 2)
    h, w = s["h"].detach(), s["w"].detach()
    return [_pick(z, lse, s["ids"]), entropy, (d @ w.float()).to(h.dtype), (d.t() @ h.float()).to(w.dtype)]


def _plain_balance(s):
    e, k, layers = s["experts"], s["k"], len(s["logits"])
    n = s["tokens"]
    m = torch.ones(n, device="cuda") if s["mask"] is None else (s["mask"] != 0).float()
    if s["cu"] is None:
        rows, seq = 1, torch.zeros(n, dtype=torch.int64, device="cuda")
    else:
        rows = s["cu"].numel() - 1
        seq = torch.searchsorted(s["cu"][1:].contiguous(), torch.arange(n, device="cuda", dtype=torch.int32), right=True)
    t = torch.zeros(rows, device="cuda").index_add_(0, seq, m)
    weight = torch.where(t > 0, e / (k * t * t), torch.zeros_like(t)) / ((t > 0).sum().clamp(min=1) * layers)
    loss = torch.zeros((), device="cuda")
    counts, grads = [], []
    for i, logits in enumerate(s["logits"]):
        x = logits.detach().float()
        if s["score"] == "softmax":
            ex = torch.exp(x - x.max(1, keepdim=True).values)
            p = ex / ex.sum(1, keepdim=True)
            slope = p
        else:
            sig = 1.0 / (1.0 + torch.exp(-x))
            p = sig / sig.sum(1, keepdim=True)
            slope = p * (1.0 - sig)
        ids = _largest(x, k) if s["ids"] is None else s["ids"][i]
        chosen = torch.zeros_like(x).scatter_add_(1, ids, torch.ones_like(ids, dtype=x.dtype)) * m[:, None]
        c = torch.zeros(rows, e, device="cuda").index_add_(0, seq, chosen)
        prob = torch.zeros(rows, e, device="cuda").index_add_(0, seq, p * m[:, None])
        loss = loss + (weight * (c * prob).sum(1)).sum()
        counts.append(c.sum(0).to(torch.int64))
        wc = (weight[:, None] * c)[seq]
        grads.append((s["g_loss"] * m[:, None] * slope * (wc - (p * wc).sum(1, keepdim=True))).to(logits.dtype))
    return [loss, torch.stack(counts)] + grads


# --------------------------------------------------------------------------------------------------------------
# the calls that a user makes
# --------------------------------------------------------------------------------------------------------------

def _own_top(s):
    from axon_amd.utils.torch.ops import top_logprobs_from_logits

    r = top_logprobs_from_logits(s["logits"], s["k"], s["labels"])
    out = [r.entropy.detach(), r.top_logprobs.detach(), r.top_ids]
    outputs, upstream = [r.entropy, r.top_logprobs], [s.get("g_en"), s.get("g_top")]
    if s["labels"] is not None:
        out.append(r.logprobs.detach())
        outputs, upstream = outputs + [r.logprobs], upstream + [s.get("g_lp")]
    if s["grad"]:
        out += torch.autograd.grad(outputs, s["logits"], upstream)
    return out


def _own_tokens(s):
    from axon_amd.utils.torch.ops import token_logprobs_from_logits

    lp, entropy = token_logprobs_from_logits(s["logits"], s["ids"])
    grad, = torch.autograd.grad([lp, entropy], s["logits"], [s["g_ids"], s["g_en"]])
    return [lp.detach(), entropy.detach(), grad]


def _own_head_top(s):
    from axon_amd.utils.kernel.linear_top_logprobs import linear_top_logprobs

    with torch.no_grad():
        r = linear_top_logprobs(s["h"], s["w"], s["k"], s["labels"], s["temperature"], s["softcap"] or None)
    return [r.entropy, r.top_logprobs, r.top_ids, r.logprobs]


def _own_head_tokens(s):
    from axon_amd.utils.kernel.linear_top_logprobs import linear_token_logprobs

    lp, entropy = linear_token_logprobs(s["h"], s["w"], s["ids"], s["temperature"], s["softcap"] or None)
    grads = torch.autograd.grad([lp, entropy], [s["h"], s["w"]], [s["g_ids"], s["g_en"]])
    return [lp.detach(), entropy.detach(), *grads]


def _own_balance(s):
    from axon_amd.trainer.algos.loss.balance import router_balance_loss

    loss, counts = router_balance_loss(s["logits"], s["k"], token_mask=s["mask"], cu_seqlens=s["cu"],
                                       expert_ids=s["ids"], score_fn=s["score"])
    return [loss.detach(), counts, *torch.autograd.grad(loss, s["logits"], s["g_loss"])]


def run(state):
    plain = dict(top=_plain_top, tokens=_plain_tokens, head_top=_plain_head_top, head_tokens=_plain_head_tokens,
                 balance=_plain_balance)
    calls = dict(top=_own_top, tokens=_own_tokens, head_top=_own_head_top, head_tokens=_own_head_tokens,
                 balance=_own_balance)
    return (calls if own else plain)[state["kind"]](state)


# --------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------

def work(case):
    kind, n = case["kind"], case["tokens"]
    if kind == "balance":
        cells = case["layers"] * n * case["experts"]
        ids = case["layers"] * n * case["k"] * 8 if case["given"] else 0
        return {"bytes": 2 * cells * (case["bits"] // 8) + ids + n * case["mask_bits"] // 8, "flops": 20.0 * cells}
    v, k = case["vocab"], case["k"]
    if kind in ("top", "tokens"):
        grad = kind == "tokens" or case["grad"]
        rows = n * v * (case["bits"] // 8)
        # alternatives: ids and log-probabilities; their gradients; the label's and the entropy's
        small = n * (12 * k + 16) + (n * (4 * k + 8) if grad else 0)
        return {"bytes": rows * (2 if grad else 1) + small, "flops": (12.0 if grad else 6.0) * n * v}
    operands = 2 * case["hidden"] * (n + v)
    if kind == "head_top":
        return {"bytes": operands + n * (12 * k + 16), "flops": 2.0 * n * case["hidden"] * v}
    return {"bytes": 2 * operands + n * (16 * k + 8), "flops": 6.0 * n * case["hidden"] * v}


# --------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------

def _exact_rows(z, ids, g_ids, g_entropy):
    """For rows of 64-bit logits: log-softmax, entropy, log-probabilities of ids and, with upstream gradients, the
    gradient of the logits."""
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    plogp = torch.special.entr(p)
    entropy = plogp.sum(1)
    ids_in = ids.clamp(0, z.shape[1] - 1)
    inside = ids_in == ids
    lp = log_p.gather(1, ids_in).masked_fill(~inside, 0.0)
    grad = None
    if g_ids is not None:
        up = g_ids.double() * inside
        grad = torch.zeros_like(z).scatter_add_(1, ids_in, up)
        grad -= up.sum(1, keepdim=True) * p
        grad += g_entropy.double()[:, None] * (plogp - p * entropy[:, None])
    return entropy, lp, grad


def _exact_order(z, k):
    return torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]


def _chunks(s, n):
    step = max(1, (1 << 28) // s["vocab"])
    return [slice(a, min(a + step, n)) for a in range(0, n, step)]


def _exact_top(s):
    n, parts = s["tokens"], []
    for c in _chunks(s, n):
        z = s["logits"].detach()[c].double()
        top = _exact_order(z, s["k"])
        ids = top if s["labels"] is None else torch.cat([top, s["labels"][c, None]], 1)
        g = None
        if s["grad"]:
            g = s["g_top"][c] if s["labels"] is None else torch.cat([s["g_top"][c], s["g_lp"][c, None]], 1)
        entropy, lp, grad = _exact_rows(z, ids, g, s["g_en"][c] if s["grad"] else None)
        parts.append([entropy, lp[:, : s["k"]], top] + ([lp[:, -1]] if s["labels"] is not None else [])
                     + ([grad] if s["grad"] else []))
    return [torch.cat(x) for x in zip(*parts)]


def _exact_tokens(s):
    parts = []
    for c in _chunks(s, s["tokens"]):
        entropy, lp, grad = _exact_rows(s["logits"].detach()[c].double(), s["ids"][c], s["g_ids"][c], s["g_en"][c])
        parts.append([lp, entropy, grad])
    return [torch.cat(x) for x in zip(*parts)]


def _exact_head(s):
    h, w = s["h"].detach().double(), s["w"].detach().double()
    cap, inv_t = s["softcap"], 1.0 / s["temperature"]
    top = s["kind"] == "head_top"
    parts, d_w = [], None if top else torch.zeros_like(w)
    for c in _chunks(s, s["tokens"]):
        raw = torch.mm(h[c], w.t())
        bent = torch.tanh(raw / cap) if cap else None
        z = (cap * bent if cap else raw) * inv_t
        if top:
            best = _exact_order(raw, s["k"])
            entropy, lp, _ = _exact_rows(z, torch.cat([best, s["labels"][c, None]], 1), None, None)
            parts.append([entropy, lp[:, :-1], best, lp[:, -1]])
            continue
        entropy, lp, d = _exact_rows(z, s["ids"][c], s["g_ids"][c], s["g_en"][c])
        d = d * inv_t
        if cap:
            d = d * (1.0 - bent * bent)
        d_w.addmm_(d.t(), h[c])
        parts.append([lp, entropy, torch.mm(d, w)])
    out = [torch.cat(x) for x in zip(*parts)]
    return out if top else out + [d_w]


def _exact_balance(s):
    n, e, k, layers = s["tokens"], s["experts"], s["k"], len(s["logits"])
    keep = torch.ones(n, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"] != 0
    bounds = [0, n] if s["cu"] is None else s["cu"].tolist()
    spans = [(a, b, float(keep[a:b].sum())) for a, b in zip(bounds[:-1], bounds[1:])]
    spans = [x for x in spans if x[2] > 0]
    loss, counts, grads = torch.zeros((), dtype=torch.float64, device="cuda"), [], []
    for i, logits in enumerate(s["logits"]):
        x = logits.detach().double().requires_grad_(True)
        score = torch.softmax(x, 1) if s["score"] == "softmax" else torch.sigmoid(x)
        if s["score"] != "softmax":
            score = score / score.sum(1, keepdim=True)
        ids = _exact_order(x.detach(), k) if s["ids"] is None else s["ids"][i]
        hits = torch.nn.functional.one_hot(ids, e).sum(1) * keep[:, None]
        layer = torch.zeros((), dtype=torch.float64, device="cuda")
        for a, b, t in spans:
            f = hits[a:b].sum(0).double() * (e / (k * t))
            layer = layer + (f * (score[a:b] * keep[a:b, None]).sum(0) / t).sum()
        layer = layer / (max(len(spans), 1) * layers)
        if spans:
            grads.append(torch.autograd.grad(layer, x)[0] * s["g_loss"].double())
        else:
            grads.append(torch.zeros_like(x))
        loss = loss + layer.detach()
        counts.append(hits.sum(0))
    return [loss, torch.stack(counts)] + grads


def exact(case, seed):
    s = prepare(case, seed)
    return dict(top=_exact_top, tokens=_exact_tokens, head_top=_exact_head, head_tokens=_exact_head,
                balance=_exact_balance)[case["kind"]](s)
