"""Plain 64-bit forms of the operators of a policy step, written out from their definitions: decode over shared pages, policy and preference losses (with what bounds their errors)."""
import math
import random

import torch


def attention(q, k, v, table, lens):
    """``[B, Hq, D]`` in 64 bits, and per element the largest value that its head meets."""
    B, hq, D = q.shape
    hkv, bs = k.shape[2], k.shape[1]
    out, top = torch.zeros(B, hq, D, dtype=torch.float64), torch.zeros(B, hq, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pages = table[b, :(n + bs - 1) // bs].long()
        kk, vv = (x[pages].reshape(-1, hkv, D)[:n].double().cpu() for x in (k, v))
        for h in range(hq):
            g = h // (hq // hkv)
            w = torch.softmax(kk[:, g] @ q[b, h].double().cpu() / math.sqrt(D), 0)
            out[b, h], top[b, h] = w @ vv[:, g], vv[:, g].abs().amax(0)
    return out, top


def batch(sizes, prompts, answers, bs, hq, hkv, D, seed=0, device='cpu', dtype=torch.bfloat16, fill=0):
    """Sequences of groups whose prompts share whole pages: ``q, k, v, table, lens, shared pages per group``; pages lie anywhere, page 0 belongs to nobody."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    shared = [p // bs for p in prompts]
    rows = [(i, prompts[i] + (rng.randint(0, answers) if answers else 0)) for i, n in enumerate(sizes) for _ in range(n)]
    own = [(n + bs - 1) // bs - shared[i] for i, n in rows]
    free = list(range(1, 1 + sum(shared) + sum(own)))
    pages = len(free) + 1
    rng.shuffle(free)
    common = [[free.pop() for _ in range(n)] for n in shared]
    lists = [common[i] + [free.pop() for _ in range(o)] for (i, _), o in zip(rows, own)] + [[]] * fill
    table = torch.zeros(len(lists), max(1, max(map(len, lists))), dtype=torch.int32)
    for r, l in zip(table, lists):
        r[:len(l)] = torch.tensor(l, dtype=torch.int32)
    lens = torch.tensor([n for _, n in rows] + [0] * fill, dtype=torch.int32)
    q = (1.5 * torch.randn(len(lists), hq, D, generator=g)).to(dtype)
    k, v = (torch.randn(pages, bs, hkv, D, generator=g).to(dtype) for _ in range(2))
    return (q.to(device), k.to(device), v.to(device), table.to(device), lens.to(device)), list(sizes) + [1] * fill, shared + [0] * fill


def policy(logps, labels, adv, old=None, ref=None, ent=None, ratio='token', surrogate='clip', reduce='sequence', epsilon=0.2, epsilon_high=None, beta=0.0, entropy_coef=0.0,
           tau=(1.0, 1.0), denominator=1.0, ignore_index=-100):
    """Loss, figures, gradients by log-probs and entropies in 64 bits, and bounds: the loss's with every term positive, the gradient's likewise."""
    mask = labels if labels.dtype == torch.bool else labels != ignore_index
    B, S = logps.shape
    hi, lo = 1 + (epsilon if epsilon_high is None else epsilon_high), 1 - epsilon
    counts, total = [int(m.sum()) for m in mask], int(mask.sum())
    loss = size = kl = low = high = 0.0
    grad, gsize, gent = (torch.zeros(B, S, dtype=torch.float64) for _ in range(3))
    for b in range(B):
        at = [t for t in range(S) if mask[b, t]]
        if not at:
            continue
        w = 1 / (B * counts[b]) if reduce == 'sequence' else 1 / (total if reduce == 'token' else denominator)
        raw = [float(logps[b, t]) - float(old[b, t]) if old is not None else 0.0 for t in at]
        lr = [min(max(x, -20.0), 20.0) for x in raw]
        if ratio == 'sequence':
            lr = [sum(lr) / len(at)] * len(at)
        by_ratio, of_ratio = [], []
        for t, l in zip(at, lr):
            r, a, lp = math.exp(l), float(adv[b] if adv.dim() == 1 else adv[b, t]), float(logps[b, t])
            direct = 0.0
            if surrogate == 'clip':
                c = min(max(r, lo), hi)
                f = -min(r * a, c * a)
                d = -r * a if r * a <= c * a else 0.0
            elif surrogate == 'soft':
                tt = tau[0] if a > 0 else tau[1]
                s = 1 / (1 + math.exp(-tt * (r - 1)))
                f, d = -s * 4 / tt * a, -4 * s * (1 - s) * r * a
            else:
                f, d, direct = -min(r, 1 + epsilon) * a * lp, 0.0, -min(r, 1 + epsilon) * a
            by_ratio.append(d)
            size_t, g_t = abs(f), abs(direct)
            of_ratio.append(abs(r * a))
            if ref is not None and beta > 0:
                x = float(ref[b, t]) - lp
                f += beta * (math.exp(x) - x - 1)
                size_t += beta * (math.exp(x) - x - 1)
                direct -= beta * math.expm1(x)
                g_t += beta * abs(math.expm1(x))
            if entropy_coef:
                f -= entropy_coef * float(ent[b, t])
                size_t += entropy_coef * float(ent[b, t])
                gent[b, t] = -entropy_coef * w
            loss, size = loss + w * f, size + w * size_t
            grad[b, t], gsize[b, t] = w * direct, w * g_t
            kl, low, high = kl + math.exp(l) - 1 - l, low + (r < lo), high + (r > hi)
        for i, t in enumerate(at):
            # of a sequence's ratio a token has the row's mean derivative w Σ d / n, whose error is bounded by w Σ |d| / n whatever the token's own term is
            d, e = (sum(by_ratio) / len(at), sum(of_ratio) / len(at)) if ratio == 'sequence' else (by_ratio[i], of_ratio[i])
            grad[b, t] += w * d * (abs(raw[i]) <= 20)
            gsize[b, t] += w * e
    n = max(total, 1)
    return dict(loss=loss, size=size, stats=[kl / n, low / n, high / n, total], grad=grad, gsize=gsize, gent=gent)


def preference(logps, labels, ref=None, form='sigmoid', beta=0.1, gamma=0.0, label_smoothing=0.0, nll_weight=0.0, ignore_index=-100):
    """Loss by its definition in 64 bits as a function of the log-probs (differentiable)."""
    mask = labels if labels.dtype == torch.bool else labels != ignore_index
    rows = [torch.where(m, x, torch.zeros_like(x)).sum() for m, x in zip(mask, logps)]
    n = [max(1, int(m.sum())) for m in mask]
    if form in ('simpo', 'orpo'):
        level = [r / k for r, k in zip(rows, n)]
    else:
        away = [0.0] * len(rows) if ref is None else [x if ref.dim() == 1 else torch.where(m, x, torch.zeros_like(x)).sum() for m, x in zip(mask, ref)]
        level = [r - a for r, a in zip(rows, away)]
    log_sigmoid = lambda z: -torch.log1p(torch.exp(-z)) if float(z.detach()) > 0 else z - torch.log1p(torch.exp(z))  # noqa: E731
    each = []
    for c, r in zip(level[0::2], level[1::2]):
        z = beta * (c - r) - gamma
        if form in ('sigmoid', 'simpo'):
            each.append(-(1 - label_smoothing) * log_sigmoid(z) - label_smoothing * log_sigmoid(-z))
        elif form == 'hinge':
            each.append(torch.clamp(1 - z, min=0))
        elif form == 'ipo':
            each.append((z - 1 / (2 * beta))**2)
        elif form == 'kto_pair':
            each.append(1 - torch.sigmoid(beta * c) + torch.sigmoid(beta * r))
        else:
            odds = c - r - torch.log(-torch.expm1(c)) + torch.log(-torch.expm1(r))
            each.append(-beta * log_sigmoid(odds))
    loss = torch.stack(each).mean()
    if nll_weight:
        loss = loss - nll_weight * torch.stack(rows[0::2]).sum() / max(1, int(mask[0::2].sum()))
    return loss
