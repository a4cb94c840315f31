"""Controls of logits by their definition, row by row in 64 bits, on the CPU."""

import math

import torch


def spans_of(lens, positions):
    """(sequence, begin, end) of every row's history."""
    out, at = [], 0
    for i, n in enumerate(lens):
        out += [(i, at, at + n)] if positions == "last" else [(i, at, p + 1) for p in range(at, at + n)]
        at += n
    return out


def of_sequence(x, i):
    return float(x[i]) if isinstance(x, torch.Tensor) else float(x)


def controlled(z, spans, tokens, *, own=None, repetition=1.0, frequency=0.0, presence=0.0, bias_ids=None, bias=None,
               keep=None, temperature=1.0):
    """(out, d out / d z, size of what has been added up) for logits ``z`` [rows, vocab]; ``keep``: truth values."""
    z = z.detach().double().cpu()
    n, v = z.shape
    out, slope, size = z.clone(), torch.ones_like(z), z.abs()
    tokens = None if tokens is None else tokens.cpu().tolist()
    own = None if own is None else (own.cpu() != 0).tolist()
    for row, (i, a, b) in enumerate(spans):
        r, f, p, t = (of_sequence(x, i) for x in (repetition, frequency, presence, temperature))
        y, s, g = out[row], slope[row], size[row]
        if tokens is not None:
            history = [(tokens[k], own is None or own[k]) for k in range(a, b) if 0 <= tokens[k] < v]
            for j in {k for k, _ in history}:
                factor = 1.0 / r if y[j] > 0 else r
                y[j] *= factor
                s[j] = factor
            g.copy_(torch.maximum(g, y.abs()))
            count = {}
            for k, mine in history:
                if mine:
                    count[k] = count.get(k, 0) + 1
            for j, c in count.items():
                y[j] -= f * c + p
                g[j] += abs(f) * c + abs(p)
        if bias is not None:
            ids, values = (bias_ids[i], bias[i]) if bias.dim() == 2 else (bias_ids, bias)
            for j, x in zip(ids.tolist(), values.tolist()):
                if 0 <= j < v:
                    y[j] += x
                    g[j] += abs(x)
        if keep is not None and keep[row] is not None:
            y[~keep[row].cpu()] = -math.inf
        s[y == -math.inf] = 0.0
        s /= t
        y /= t
        g /= t
    return out, slope, size


def scored(out, slope, labels, g_lp=None, g_ent=None):
    """(log-probabilities, entropy, gradient of the logits, size of its terms) from controlled logits in 64 bits."""
    alive = (out > -math.inf).any(1, keepdim=True) | torch.isnan(out).any(1, keepdim=True)
    log_p = torch.log_softmax(torch.where(alive, out, torch.zeros_like(out)), 1)
    log_p = torch.where(alive, log_p, torch.full_like(log_p, -math.inf))
    p = log_p.exp()
    plogp = torch.where(p == 0, torch.zeros_like(p), p * log_p)
    entropy = -plogp.sum(1)
    v = out.shape[1]
    labels = labels.cpu().long()
    ok = (labels >= 0) & (labels < v)
    at = torch.where(ok, labels, torch.zeros_like(labels))[:, None]
    lp = torch.where(ok, log_p.gather(1, at).squeeze(1), torch.zeros(len(labels), dtype=torch.float64))
    if g_lp is None:
        return lp, entropy
    g = torch.where(ok, g_lp.double().cpu(), torch.zeros(len(labels), dtype=torch.float64))[:, None]
    ge = g_ent.double().cpu()[:, None]
    hit = torch.zeros_like(out).scatter_(1, at, g)
    grad = (hit - p * g - ge * (plogp + p * entropy[:, None])) * slope
    size = (hit.abs() + p * g.abs() + ge.abs() * (plogp.abs() + p * (entropy[:, None] + 1))) * slope
    return lp, entropy, torch.where(slope == 0, torch.zeros_like(grad), grad), size


def pack(keep):
    """int32 bit masks of truth values [rows, vocab]."""
    rows, v = keep.shape
    bits = torch.nn.functional.pad(keep.long(), (0, -v % 32)).view(rows, -1, 32)
    words = (bits << torch.arange(32, device=keep.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
