"""Sampling controls of logits and distillation from a teacher's top tokens: what is measured of them.

Each case is one pass through one operator as a user's program calls it: a decoder that penalises repeated tokens and
applies biases and a grammar to the logits of the tokens that it is about to sample, a trainer that needs the
log-probabilities of a rollout under the distribution that it was drawn from (alone, or forward and backward), and a
student that is trained on the tokens and log-probabilities that a teacher has stored, forward and backward.

``run`` computes the operators in plain torch operations in 32 bits where ``own`` is false, and calls the package where
it is true.  ``exact`` states the same definitions in 64 bits.  All inputs are synthetic and made on the GPU from the
seed.

Definitions.  Controls: a row's history is its sequence's tokens up to the row's own position, its own tokens are those
of them that the model has generated.  ``y = z / r`` where a token of the history has ``z > 0``, ``z r`` where not; minus
``f`` times how often it is among the own tokens, minus ``a`` if it is; plus its bias; ``-inf`` where the grammar's bit is
0; over the temperature.  Log-probabilities and entropy are those of ``softmax(y)``; a row that nothing is left of has
log-probability ``-inf``, entropy 0 and no gradient.  Distillation: with ``q`` the teacher's probabilities of the given
tokens and ``p`` the student's (softmax over the whole vocabulary, at a temperature), forward ``sum q log(q/p)``, reverse
``sum p log(p/q)``, or ``b sum q log(q/m) + (1-b) sum p log(p/m)`` with ``m = b q + (1-b) p``; over the given tokens
alone, or with what is left of both as one more outcome, or with the teacher's renormalised over the given tokens.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # set by the program that imports this file

VOCABS = (151936, 201088, 32768, 50257)

MAX_LOGITS = 4096 * 151936
MAX_PAIRS = 16 << 20  # tokens of all rows' histories together


def listed():
    return [
        # A decoder's single sequence under all penalties, no grammar: latency.
        dict(name="controls_one_token", kind="controls", rows=1, vocab=151936, bits=16, history=900, repetition=1.15,
             frequency=0.2, presence=0.3, biases=0, grammar="none", temperature=0.7),
        # A decode batch with long histories, per-request biases and a grammar, fp32 logits, an odd number of rows.
        dict(name="controls_decode_batch", kind="controls", rows=61, vocab=201088, bits=32, history=4000, repetition=1.1,
             frequency=0.1, presence=0.0, biases=300, grammar="states", temperature=1.0),
        # A large batch on a small vocabulary, repetition penalty and one mask for all.
        dict(name="controls_large_batch", kind="controls", rows=1024, vocab=32768, bits=16, history=1500, repetition=1.2,
             frequency=0.0, presence=0.0, biases=0, grammar="shared", temperature=1.0),
        # A short response scored under a grammar and trained on: with the gradient.
        dict(name="scored_short_grad", kind="scored", tokens=187, vocab=151936, bits=16, length=90, repetition=1.0,
             frequency=0.0, presence=0.0, biases=0, grammar="states", temperature=1.0, grad=True),
        # The old log-probabilities of a micro-batch that was sampled with every control there is.
        dict(name="scored_micro_batch", kind="scored", tokens=4096, vocab=151936, bits=16, length=900, repetition=1.1,
             frequency=0.2, presence=0.1, biases=40, grammar="states", temperature=0.8, grad=False),
        # Penalties alone on an odd vocabulary whose rows start off every boundary: with the gradient.
        dict(name="scored_odd_vocab_grad", kind="scored", tokens=2047, vocab=50257, bits=16, length=400, repetition=1.3,
             frequency=0.3, presence=0.5, biases=0, grammar="none", temperature=1.0, grad=True),
        # Long sequences, fp32 logits, repetition penalty: with the gradient.
        dict(name="scored_long_grad", kind="scored", tokens=1500, vocab=151936, bits=32, length=1500, repetition=1.1,
             frequency=0.0, presence=0.0, biases=0, grammar="none", temperature=1.0, grad=True),
        # A student's losses on a short response, weighed by the caller afterwards: latency.
        dict(name="distill_short", kind="distill", tokens=61, vocab=151936, bits=16, k=8, divergence="forward",
             tail="drop", beta=0.5, temperature=1.0, weighted=False, masked=0.0),
        # A student's step on a packed micro-batch, a third of it prompt, with what the teacher left out as one outcome.
        dict(name="distill_micro_batch", kind="distill", tokens=4096, vocab=151936, bits=16, k=64, divergence="forward",
             tail="rest", beta=0.5, temperature=1.0, weighted=True, masked=0.33),
        # On-policy distillation (reverse) of a whole micro-batch on the largest vocabulary.
        dict(name="distill_reverse", kind="distill", tokens=2500, vocab=201088, bits=16, k=20, divergence="reverse",
             tail="rest", beta=0.5, temperature=1.0, weighted=True, masked=0.0),
        # The generalised Jensen-Shannon divergence on fp32 logits.
        dict(name="distill_jsd", kind="distill", tokens=1500, vocab=151936, bits=32, k=32, divergence="jsd",
             tail="renormalize", beta=0.3, temperature=2.0, weighted=True, masked=0.0),
        # An odd vocabulary, weighed by the caller afterwards.
        dict(name="distill_odd_vocab", kind="distill", tokens=2047, vocab=50257, bits=16, k=128, divergence="forward",
             tail="renormalize", beta=0.5, temperature=1.0, weighted=False, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; counts are spread over their logarithm."""
    kind = rng.choice(("controls", "scored", "distill"))
    vocab = rng.choice(VOCABS + (_log_int(rng, 1000, 260000),))
    bits = rng.choice((16, 16, 32))
    if kind == "distill":
        tokens = _log_int(rng, 1, max(2, min(8192, MAX_LOGITS // (vocab * bits // 16))))
        return dict(kind=kind, tokens=tokens, vocab=vocab, bits=bits, k=_log_int(rng, 1, 128),
                    divergence=rng.choice(("forward", "forward", "reverse", "jsd")),
                    tail=rng.choice(("rest", "drop", "renormalize")), beta=rng.choice((0.1, 0.5, 0.7)),
                    temperature=rng.choice((1.0, 1.0, 2.0)), weighted=rng.random() < 0.7,
                    masked=rng.choice((0.0, 0.0, 0.4)))
    c = dict(kind=kind, vocab=vocab, bits=bits, repetition=rng.choice((1.0, 1.1, 1.3, 0.9)),
             frequency=rng.choice((0.0, 0.2, -0.1)), presence=rng.choice((0.0, 0.4)),
             biases=rng.choice((0, 0, _log_int(rng, 1, 300))), grammar=rng.choice(("none", "shared", "states", "states")),
             temperature=rng.choice((1.0, 0.7, 1.3)))
    if kind == "controls":
        rows = _log_int(rng, 1, max(2, min(1024, MAX_LOGITS // (vocab * bits // 16))))
        return dict(c, rows=rows, history=_log_int(rng, 1, min(32768, MAX_PAIRS // rows)))
    grad = rng.random() < 0.6
    tokens = _log_int(rng, 1, max(2, min(8192, MAX_LOGITS // (vocab * (bits // 16) * (2 if grad else 1)))))
    return dict(c, tokens=tokens, length=_log_int(rng, 1, min(8192, MAX_PAIRS // tokens)), grad=grad)


# --------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _logits(g, n, v, at):
    """A trained model's: sure of most tokens."""
    z = torch.empty(n, v, device="cuda").normal_(0.0, 2.0, generator=g)
    z[torch.arange(n, device="cuda"), at] += 12.0 + 6.0 * torch.rand(n, generator=g, device="cuda")
    return z


def _text(g, n, v):
    """Token ids in which some come back all the time and most hardly ever."""
    return (torch.rand(n, generator=g, device="cuda") ** 4 * v).long().clamp_(max=v - 1)


def _pack_bits(keep):
    """Truth values [rows, vocab] as 32-bit words, bit i of word w for token 32 w + i."""
    rows, v = keep.shape
    bits = torch.nn.functional.pad(keep, (0, -v % 32)).view(rows, -1, 32).long()
    words = (bits << torch.arange(32, device=keep.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _grammar(c, g, r, rows, chosen):
    """What may be sampled: for all rows the same, or by the state that a grammar is in (-1: anything).  The tokens that
    were chosen are among it, but for a few rows."""
    v = c["vocab"]
    if c["grammar"] == "none":
        return None, None
    states = 1 if c["grammar"] == "shared" else min(64, rows)
    index = torch.randint(-1 if states > 1 else 0, states, (rows,), generator=g, device="cuda")
    keep = torch.rand(states, v, generator=g, device="cuda") < 0.97
    if states > 1:  # half of the states leave little: digits, a closing bracket, the keys of an object
        keep[::2] = torch.rand(-(-states // 2), v, generator=g, device="cuda") < r.choice((0.0005, 0.01))
    keep[index.clamp(min=0), chosen] = True
    if states > 1:
        keep[states - 1] = False  # nothing at all
        keep[states - 1, v // 3] = rows % 2 == 0
    return _pack_bits(keep), None if states == 1 else index.to(torch.int32)


def _lengths(total, mean, r):
    lens, left = [], total
    while left > 0:
        x = min(max(int(round(mean * math.exp(r.gauss(0.0, 0.5)))), 1), left)
        lens.append(x)
        left -= x
    return lens


def _offsets(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _prepare_controls(c, g, r):
    v, last = c["vocab"], c["kind"] == "controls"
    lens = [max(1, int(c["history"] * r.uniform(0.3, 1.0))) for _ in range(c["rows"])] if last else \
        _lengths(c["tokens"], c["length"], r)
    lens[0] = c["history"] if last else lens[0]
    total = sum(lens)
    cu, ids = _offsets(lens), _text(g, total, v)
    response = torch.rand(total, generator=g, device="cuda") < 0.0
    for a, x in zip(cu.tolist(), lens):  # a prompt, then what the model has written
        response[a + int(0.3 * x): a + x] = True
    rows = len(lens) if last else total
    labels = _text(g, rows, v) if last else torch.roll(ids, -1)
    z = _logits(g, rows, v, labels)
    dtype = torch.bfloat16 if c["bits"] == 16 else torch.float32
    s = dict(c, rows=rows, ids=ids, cu=cu, response=response.float(), labels=labels, logits=z.to(dtype))
    s["allowed"], s["index"] = _grammar(c, g, r, rows, labels)
    s["bias_ids"] = s["bias"] = None
    if c["biases"]:  # per request: a few tokens pushed up or down, one of them out; short requests filled up with -1
        k = min(c["biases"], v)
        per = len(lens) if last else 1
        s["bias_ids"] = torch.stack([torch.randperm(v, generator=g, device="cuda")[:k] for _ in range(min(per, 8))])
        s["bias_ids"] = s["bias_ids"][torch.arange(per, device="cuda") % 8] if per > 8 else s["bias_ids"]
        s["bias"] = 3.0 * _randn(g, per, k)
        if k > 2:
            s["bias"][:, 1] = -math.inf
            s["bias_ids"][::2, -1] = -1
        if per == 1:
            s["bias_ids"], s["bias"] = s["bias_ids"][0], s["bias"][0]
    if not last and c["grad"]:
        s["g_lp"] = _randn(g, rows) / rows
        s["g_en"] = -0.01 / rows + 0.001 * _randn(g, rows) / rows
        s["logits"].requires_grad_(True)
    return s


def _prepare_distill(c, g):
    n, v = c["tokens"], c["vocab"]
    k = min(c["k"], v)
    z = _logits(g, n, v, _text(g, n, v))
    # a teacher that agrees with the student in most and has its own view in the rest
    top = (z / c["temperature"] + _randn(g, n, v))
    lse = torch.logsumexp(top, 1, keepdim=True)
    best = top.topk(k, dim=1)
    ids, lq = best.indices, best.values - lse
    ids = torch.where(torch.rand(n, k, generator=g, device="cuda") < 0.01, torch.full_like(ids, -1), ids)
    s = dict(c, k=k, logits=z.to(torch.bfloat16 if c["bits"] == 16 else torch.float32).requires_grad_(True), ids=ids, lq=lq)
    keep = (torch.rand(n, generator=g, device="cuda") >= c["masked"]).float()
    keep[0] = 1.0
    s["weights"] = keep * (0.5 / n)  # a coefficient, a mask, a mean over tokens
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "distill":
        return _prepare_distill(case, g)
    return _prepare_controls(case, g, random.Random(seed))


# --------------------------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# --------------------------------------------------------------------------------------------------------------

def _histories(s):
    """(row, token) for every token of every row's history."""
    rows = torch.arange(s["rows"], device="cuda")
    cu = s["cu"].long()
    if s["kind"] == "controls":
        start, end = cu[:-1], cu[1:]
    else:
        start, end = cu[torch.searchsorted(cu, rows, right=True) - 1], rows + 1
    count = end - start
    row = torch.repeat_interleave(rows, count)
    return row, torch.arange(row.numel(), device="cuda") - (torch.cumsum(count, 0) - count)[row] + start[row]


def _plain_controlled(s):
    """(y, dy / dz) in 32 bits, before the temperature in neither."""
    z = s["logits"].detach().float()
    n, v = z.shape
    slope = torch.ones_like(z)
    row, token = _histories(s)
    at = row * v + s["ids"][token]
    if s["repetition"] != 1.0:
        seen = torch.zeros(n * v, dtype=torch.bool, device="cuda")
        seen[at] = True
        r = torch.tensor(s["repetition"], device="cuda")
        slope = torch.where(seen.view(n, v), torch.where(z > 0, 1.0 / r, r), slope)
        z = z * slope
    if s["frequency"] != 0.0 or s["presence"] != 0.0:
        count = torch.zeros(n * v, device="cuda").scatter_add_(0, at, s["response"][token]).view(n, v)
        z = z - (s["frequency"] * count + s["presence"] * (count > 0))
    if s["bias"] is not None:
        per = s["bias_ids"].dim() == 2
        ids = s["bias_ids"] if per else s["bias_ids"].expand(n, -1)
        bias = s["bias"] if per else s["bias"].expand(n, -1)
        ok = ids >= 0
        z = z.scatter_add(1, ids.clamp(min=0), torch.where(ok, bias, torch.zeros_like(bias)))
    if s["allowed"] is not None:
        words = s["allowed"] if s["index"] is None else s["allowed"][s["index"].clamp(min=0).long()]
        at = torch.arange(v, device="cuda")
        keep = ((words[:, at // 32] >> (at % 32)) & 1) != 0
        if s["index"] is not None:
            keep = keep | (s["index"] < 0)[:, None]
        z = torch.where(keep, z, torch.full_like(z, -math.inf))
    return z, torch.where(z > -math.inf, slope, torch.zeros_like(slope))


def _plain_controls(s):
    y, _ = _plain_controlled(s)
    return [(y / s["temperature"]).to(s["logits"].dtype)]


def _plain_scored(s):
    y, slope = _plain_controlled(s)
    y = y / s["temperature"]
    m = y.max(1, keepdim=True).values
    alive = m > -math.inf
    m = torch.where(alive, m, torch.zeros_like(m))
    ex = torch.exp(y - m)
    total = ex.sum(1, keepdim=True)
    log_total = torch.log(total)
    p = torch.where(alive, ex / total, torch.zeros_like(ex))
    log_p = torch.where(p > 0, (y - m) - log_total, torch.zeros_like(y))
    entropy = -(p * log_p).sum(1)
    at = s["labels"][:, None]
    lp = torch.where(alive, y.gather(1, at) - m - log_total, torch.full_like(m, -math.inf)).squeeze(1)
    out = [lp, entropy]
    if s["grad"]:
        d = -p * (s["g_lp"][:, None] + s["g_en"][:, None] * (log_p + entropy[:, None]))
        d = d.scatter_add_(1, at, s["g_lp"][:, None])
        d = torch.where(alive, d * (slope / s["temperature"]), torch.zeros_like(d))
        out.append(d.to(s["logits"].dtype))
    return out


def _outcomes(s, lq, lp, ok, divergence):
    """(terms, dL / dlp) of outcomes with the teacher's and the student's log-probabilities."""
    none = torch.zeros_like(lp)
    q = torch.where(ok, torch.exp(lq), none)
    p = torch.where(ok, torch.exp(lp), none)
    lq_, lp_ = torch.where(q > 0, lq, none), torch.where(p > 0, lp, none)
    if divergence == "forward":
        return torch.where(q > 0, q * (lq_ - lp), none), -q
    if divergence == "reverse":
        return torch.where(p > 0, p * (lp_ - lq), none), torch.where(p > 0, p * (lp_ - lq + 1.0), none)
    b = s["beta"]
    lm = torch.log(b * q + (1.0 - b) * p)
    mine = torch.where(p > 0, (1.0 - b) * p * (lp_ - lm), none)
    return torch.where(q > 0, b * q * (lq_ - lm), none) + mine, mine


def _plain_distill(s):
    z = s["logits"].detach().float() / s["temperature"]
    ids = s["ids"]
    ok = ids >= 0
    at = ids.clamp(min=0)
    m = z.max(1, keepdim=True).values
    ex = torch.exp(z - m)
    log_total = torch.log(ex.sum(1, keepdim=True))
    lp = z.gather(1, at) - m - log_total
    lq = torch.where(ok, s["lq"], torch.full_like(s["lq"], -math.inf))
    if s["tail"] == "renormalize":
        top = lq.max(1, keepdim=True).values
        top = torch.where(top > -math.inf, top, torch.zeros_like(top))
        lq = lq - top - torch.log(torch.exp(lq - top).sum(1, keepdim=True))
    terms, g = _outcomes(s, lq, lp, ok, s["divergence"])
    losses, total = terms.sum(1), g.sum(1, keepdim=True)
    covered = torch.where(ok, torch.exp(lp), torch.zeros_like(lp)).sum(1)
    p = ex / ex.sum(1, keepdim=True)
    scale = -total
    if s["tail"] == "rest":  # what is not given, summed by itself: 1 minus the rest would lose it
        given = torch.zeros(z.shape, dtype=torch.bool, device="cuda").scatter_(1, at, ok)
        given[:, 0] = (ids == 0).any(1)
        p_rest = torch.where(given, torch.zeros_like(p), p).sum(1, keepdim=True)
        q_rest = (1.0 - torch.exp(lq.double()).sum(1, keepdim=True)).clamp(min=0.0)
        t, g_rest = _outcomes(s, torch.log(q_rest).float(), torch.log(p_rest), torch.ones_like(p_rest, dtype=torch.bool),
                              s["divergence"])
        losses = losses + t.squeeze(1)
        total = total + g_rest
        scale = torch.where(given, -total, torch.where(p_rest > 0, g_rest / p_rest, torch.zeros_like(p_rest)) - total)
    d = (p * scale).scatter_add_(1, at, torch.where(ok, g, torch.zeros_like(g)))
    w = s["weights"]
    on = (w != 0) if s["weighted"] else torch.ones_like(w, dtype=torch.bool)
    losses = torch.where(on, losses, torch.zeros_like(losses))
    covered = torch.where(on, covered, torch.zeros_like(covered))
    d = (d * (w / s["temperature"])[:, None]).to(s["logits"].dtype)
    if s["weighted"]:
        return [(w * losses).sum(), losses, covered, d]
    return [losses, covered, d]


# --------------------------------------------------------------------------------------------------------------
# the calls that a user makes
# --------------------------------------------------------------------------------------------------------------

def _own_logit_controls(s, positions):
    from axon_amd.utils.torch.controls import LogitControls

    return LogitControls(s["ids"], s["cu"], positions=positions, response_mask=s["response"],
                         repetition_penalty=s["repetition"], frequency_penalty=s["frequency"],
                         presence_penalty=s["presence"], bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"],
                         allowed_index=s["index"], temperature=s["temperature"])


def _own_controls(s):
    from axon_amd.utils.torch.controls import controlled_logits

    return [controlled_logits(s["logits"], _own_logit_controls(s, "last"))]


def _own_scored(s):
    from axon_amd.utils.torch.controls import controlled_logprobs_from_logits

    lp, entropy = controlled_logprobs_from_logits(s["logits"], s["labels"], _own_logit_controls(s, "all"))
    out = [lp.detach(), entropy.detach()]
    if s["grad"]:
        out += torch.autograd.grad([lp, entropy], s["logits"], [s["g_lp"], s["g_en"]])
    return out


def _own_distill(s):
    from axon_amd.utils.torch.distillation import distillation_from_logits, distillation_loss_from_logits

    how = dict(divergence=s["divergence"], tail=s["tail"], beta=s["beta"], temperature=s["temperature"])
    if s["weighted"]:
        r = distillation_loss_from_logits(s["logits"], s["ids"], s["lq"], s["weights"], **how)
        return [r.loss.detach(), r.losses, r.covered, *torch.autograd.grad(r.loss, s["logits"])]
    losses, covered = distillation_from_logits(s["logits"], s["ids"], s["lq"], **how)
    return [losses.detach(), covered, *torch.autograd.grad(losses, s["logits"], s["weights"])]


def run(state):
    plain = dict(controls=_plain_controls, scored=_plain_scored, distill=_plain_distill)
    calls = dict(controls=_own_controls, scored=_own_scored, distill=_own_distill)
    return (calls if own else plain)[state["kind"]](state)


# --------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------

def work(case):
    v, size = case["vocab"], case["bits"] // 8
    if case["kind"] == "distill":
        n, k = case["tokens"], case["k"]
        read = n * (1.0 - case["masked"]) if case["weighted"] else n
        return {"bytes": (read + n) * v * size + n * (12 * k + 12), "flops": 12.0 * n * v}
    last = case["kind"] == "controls"
    n = case["rows"] if last else case["tokens"]
    masks = 0 if case["grammar"] == "none" else v // 8 * (1 if case["grammar"] == "shared" else min(64, n))
    tokens = int(0.65 * n * case["history"]) if last else n
    moved = 2 if last or case["grad"] else 1
    small = tokens * 12 + masks + case["biases"] * 12 * (n if last else 1) + (0 if last else 24 * n)
    return {"bytes": n * v * size * moved + small, "flops": (4.0 if last else 14.0 if case["grad"] else 8.0) * n * v}


# --------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------

def _exact_row_controls(s, r, begin, end, sequence, z):
    """A row's controlled logits, before the temperature, as a function of its logits ``z`` (64 bits)."""
    v = z.shape[0]
    ids, mine = s["ids"][begin:end], s["response"][begin:end] != 0
    if s["repetition"] != 1.0:
        seen = torch.bincount(ids, minlength=v) > 0
        z = torch.where(seen & (z > 0), z / s["repetition"], torch.where(seen, z * s["repetition"], z))
    count = torch.bincount(ids, weights=mine.double(), minlength=v)
    z = z - s["frequency"] * count - s["presence"] * (count > 0).double()
    if s["bias"] is not None:
        at, b = (s["bias_ids"][sequence], s["bias"][sequence]) if s["bias_ids"].dim() == 2 else (s["bias_ids"], s["bias"])
        z = z + torch.bincount(at.clamp(min=0), weights=torch.where(at >= 0, b.double(), 0.0), minlength=v)
    if s["allowed"] is not None:
        state = 0 if s["index"] is None else s["index_list"][r]
        if state >= 0:
            z = z.masked_fill(~s["keep"][state], -math.inf)
    return z


def _exact_controls(case, s):
    v = s["vocab"]
    if s["allowed"] is not None:
        bits = torch.arange(32, device="cuda")
        s["keep"] = ((s["allowed"].long()[:, :, None] >> bits) & 1).bool().flatten(1)[:, :v]
        s["index_list"] = None if s["index"] is None else s["index"].tolist()
    cu, last = s["cu"].tolist(), s["kind"] == "controls"
    spans = [(a, b, i) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:]))] if last else \
        [(a, p + 1, i) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])) for p in range(a, b)]
    logits, t = s["logits"].detach(), s["temperature"]
    if last:
        return [torch.stack([_exact_row_controls(s, r, a, b, i, logits[r].double()) / t for r, (a, b, i) in enumerate(spans)])]
    lps, entropies, grads = [], [], []
    labels = s["labels"].tolist()
    for r, (a, b, i) in enumerate(spans):
        z = logits[r].double().requires_grad_(s["grad"])
        with torch.enable_grad():
            log_p = torch.log_softmax(_exact_row_controls(s, r, a, b, i, z) / t, 0)
            entropy = torch.special.entr(log_p.exp()).sum()
        lps.append(log_p[labels[r]].detach())
        entropies.append(entropy.detach())
        if s["grad"]:  # by hand from log p on: where p is 0 the derivative of its logarithm is none
            p = log_p.detach().exp()
            up = -s["g_en"][r].double() * torch.where(p > 0, p * (log_p.detach() + entropy.detach()), 0.0) - s["g_lp"][r].double() * p
            up[labels[r]] += s["g_lp"][r].double()
            with torch.enable_grad():
                y = _exact_row_controls(s, r, a, b, i, z)
            grads.append(torch.autograd.grad(y, z, torch.where(torch.isfinite(y), up / t, 0.0))[0])
    lp, entropy = torch.stack(lps), torch.stack(entropies)
    dead = torch.isnan(lp)  # a row that nothing is left of
    out = [lp.masked_fill(dead, -math.inf), entropy.masked_fill(dead, 0.0)]
    return out + [torch.stack(grads)] if s["grad"] else out


def _exact_divergence(kind, beta, q, p):
    """Sum over the last dimension; an outcome that neither has counts nothing."""
    if kind == "forward":
        return (torch.special.xlogy(q, q) - torch.special.xlogy(q, p)).sum(-1)
    if kind == "reverse":
        return (torch.special.xlogy(p, p) - torch.special.xlogy(p, q)).sum(-1)
    m = beta * q + (1 - beta) * p
    m = torch.where(m > 0, m, 1.0)
    return (beta * (torch.special.xlogy(q, q) - torch.special.xlogy(q, m))
            + (1 - beta) * (torch.special.xlogy(p, p) - torch.special.xlogy(p, m))).sum(-1)


def _exact_distill(case, s):
    n, v = s["tokens"], s["vocab"]
    parts = []
    step = max(1, (1 << 27) // v)
    for c in (slice(a, min(a + step, n)) for a in range(0, n, step)):
        z = s["logits"].detach()[c].double().requires_grad_(True)
        ids = s["ids"][c]
        ok = ids >= 0
        q = torch.where(ok, s["lq"][c].double().exp(), 0.0)
        if s["tail"] == "renormalize":
            q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
        with torch.enable_grad():
            every = torch.softmax(z / s["temperature"], 1)
            p = torch.where(ok, every.gather(1, ids.clamp(min=0)), 0.0)
            covered = p.sum(1).detach()
            if s["tail"] == "rest":
                listed = torch.zeros(every.shape, device="cuda").scatter_add_(1, ids.clamp(min=0), ok.float()) > 0
                p = torch.cat([p, every.masked_fill(listed, 0.0).sum(1, keepdim=True)], 1)
                q = torch.cat([q, (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0)], 1)
            losses = _exact_divergence(s["divergence"], s["beta"], q, p)
        w = s["weights"][c].double()
        grad = torch.autograd.grad(losses, z, w)[0]
        on = (w != 0).double() if s["weighted"] else torch.ones_like(w)
        parts.append([losses.detach() * on, covered * on, grad])
    out = [torch.cat(x) for x in zip(*parts)]
    return [(out[0] * s["weights"].double()).sum(), *out] if s["weighted"] else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "distill":
        return _exact_distill(case, s)
    if case["kind"] == "scored" and s["rows"] * s["vocab"] > 2 * MAX_LOGITS:
        return None
    return _exact_controls(case, s)
