"""Operators of a group-relative policy step, from the group's prompt to its gradient.

A policy step samples several answers to every prompt and trains on the groups.  What the answers of a group have in common is kept and read once:

``attend``  one token for every sequence against the paged cache where groups of sequences share the pages of their prompt
            (``ops.paged_attention_shared`` with the plan that a decode loop keeps, ``ops.shared_prefix``)
``copy``    pages of all layers' pools in one go (``ops.cache_copy``): forks take a copy of the page that their prompt ends in, compaction moves
            whole pages
``policy``  the clipped policy loss of a batch with its KL and entropy terms, forward and backward (``ops.policy_loss``)
``prefer``  the paired loss of a preference batch, forward and backward (``ops.preference_loss``)

Widths are those of the presets ``qwen3-0.6b`` (16 / 8 heads of 128, 28 layers), ``qwen3-8b`` (32 / 8) and ``qwen3-30b-a3b`` (32 / 4); pages hold
16 tokens unless a case says otherwise.
"""
from __future__ import annotations

import math
import random
import zlib

import torch

#: Where false, ``run`` computes in elementary torch operations; where true, it calls the framework's operators.
own = False

_FORMS = ('sigmoid', 'hinge', 'ipo', 'kto_pair', 'simpo', 'orpo')


def listed():
    return [
        # four answers to one short question on a small model: a step is a few launches
        {'name': 'attend-short', 'kind': 'attend', 'sizes': '4', 'prompts': '509', 'answer': 64, 'heads': 16, 'kv_heads': 8, 'dim': 128, 'block': 16, 'fill': 0},
        # a policy step's rollout: eight questions, eight answers each, half way through
        {'name': 'attend-rollout', 'kind': 'attend', 'sizes': '8,8,8,8,8,8,8,8', 'prompts': '1024,1531,700,2048,1290,911,1777,1183', 'answer': 1024,
         'heads': 32, 'kv_heads': 8, 'dim': 128, 'block': 16, 'fill': 0},
        # answers to a question about a long document, three of sixteen finished: the batch is filled up to a power of two
        {'name': 'attend-document', 'kind': 'attend', 'sizes': '13', 'prompts': '32751', 'answer': 512, 'heads': 32, 'kv_heads': 4, 'dim': 128, 'block': 16, 'fill': 3},
        # a system prompt with examples in front of every sequence of a batch
        {'name': 'attend-system', 'kind': 'attend', 'sizes': '128', 'prompts': '8192', 'answer': 384, 'heads': 32, 'kv_heads': 8, 'dim': 128, 'block': 16, 'fill': 0},
        # one prompt of a small model forks into eight
        {'name': 'copy-fork', 'kind': 'copy', 'mode': 'fork', 'prompts': 1, 'samples': 8, 'layers': 28, 'kv_heads': 8, 'width': 128, 'value': 128, 'block': 16, 'pages': 256,
         'type': 'bf16'},
        # the prompts of a rollout fork into sixteen each
        {'name': 'copy-rollout', 'kind': 'copy', 'mode': 'fork', 'prompts': 16, 'samples': 16, 'layers': 28, 'kv_heads': 8, 'width': 128, 'value': 128, 'block': 16, 'pages': 700,
         'type': 'bf16'},
        # what is alive moves to the front of the pools, whose tail is then given back
        {'name': 'copy-compact', 'kind': 'copy', 'mode': 'compact', 'prompts': 420, 'samples': 0, 'layers': 28, 'kv_heads': 8, 'width': 128, 'value': 128, 'block': 16,
         'pages': 1024, 'type': 'bf16'},
        # a micro-batch of one group
        {'name': 'policy-micro', 'kind': 'policy', 'rows': 8, 'cols': 1024, 'ratio': 'token', 'surrogate': 'clip', 'reduce': 'sequence', 'beta': 0.0, 'entropy': 0.0,
         'advantage': 'row', 'old': True},
        # the batch of a step with a reference policy and an entropy bonus
        {'name': 'policy-step', 'kind': 'policy', 'rows': 64, 'cols': 4095, 'ratio': 'token', 'surrogate': 'clip', 'reduce': 'token', 'beta': 0.04, 'entropy': 0.01,
         'advantage': 'token', 'old': True},
        # long answers with sequence ratios
        {'name': 'policy-sequence', 'kind': 'policy', 'rows': 256, 'cols': 16384, 'ratio': 'sequence', 'surrogate': 'clip', 'reduce': 'sequence', 'beta': 0.04, 'entropy': 0.0,
         'advantage': 'row', 'old': True},
        # two pairs of answers
        {'name': 'prefer-micro', 'kind': 'prefer', 'rows': 4, 'cols': 2047, 'form': 'sigmoid', 'reference': 'token', 'smoothing': 0.0, 'nll': 0.0},
        # a large batch of pairs, with the likelihood of the chosen answers beside it
        {'name': 'prefer-batch', 'kind': 'prefer', 'rows': 512, 'cols': 8192, 'form': 'sigmoid', 'reference': 'token', 'smoothing': 0.1, 'nll': 0.2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['attend', 'attend', 'copy', 'policy', 'prefer'])
    if kind == 'attend':
        heads = rng.choice([(16, 8), (32, 8), (32, 4), (28, 4), (12, 2)])
        n = _log(rng, 1, 128)
        sizes = []
        while sum(sizes) < n:
            sizes.append(min(n - sum(sizes), _log(rng, 1, 64)))
        prompts = [_log(rng, 8, max(16, 32768 // len(sizes))) for _ in sizes]
        return {'kind': kind, 'sizes': ','.join(map(str, sizes)), 'prompts': ','.join(map(str, prompts)), 'answer': _log(rng, 1, max(2, min(1024, 65536 // n))),
                'heads': heads[0], 'kv_heads': heads[1], 'dim': rng.choice([64, 128, 128]), 'block': rng.choice([8, 16, 16, 32, 64]), 'fill': rng.choice([0, 0, 1, 5])}
    if kind == 'copy':
        mode, kv = rng.choice(['fork', 'fork', 'compact']), rng.choice([1, 2, 4, 8])
        width = rng.choice([64, 128, 128, 80])
        case = {'kind': kind, 'mode': mode, 'layers': rng.randint(1, 28), 'kv_heads': kv, 'width': width, 'value': rng.choice([width, 64]), 'block': rng.choice([8, 16, 32]),
                'type': rng.choice(['bf16', 'bf16', 'fp32'])}
        if mode == 'fork':
            prompts = _log(rng, 1, 12)
            samples = _log(rng, 2, 16)
            pages = prompts * samples + rng.randint(8, 64)
        else:
            pages = _log(rng, 8, 256)
            prompts, samples = rng.randint(1, pages // 2 - 1), 0
        case.update(prompts=prompts, samples=samples, pages=pages)
        return case
    rows, cols = 2 * _log(rng, 1, 128), _log(rng, 1, 16384)
    cols = min(cols, 4194304 // rows)
    if kind == 'policy':
        ratio, surrogate = rng.choice([('token', 'clip'), ('token', 'clip'), ('sequence', 'clip'), ('token', 'soft'), ('token', 'weight')])
        return {'kind': kind, 'rows': rows - rng.randint(0, 1), 'cols': cols, 'ratio': ratio, 'surrogate': surrogate, 'reduce': rng.choice(['sequence', 'token', 'sum']),
                'beta': rng.choice([0.0, 0.04, 0.2]), 'entropy': rng.choice([0.0, 0.0, 0.01]), 'advantage': rng.choice(['row', 'token']), 'old': rng.random() < 0.9}
    return {'kind': kind, 'rows': rows, 'cols': cols, 'form': rng.choice(_FORMS), 'reference': rng.choice(['token', 'row', 'none']), 'smoothing': 0.0,
            'nll': rng.choice([0.0, 0.2])}


# ------------------------------------------------------------------- inputs
def _gen(seed, name):
    return torch.Generator(device='cuda').manual_seed((zlib.crc32(name.encode()) << 20) + int(seed) % (1 << 20))


def _ints(text):
    return [int(x) for x in text.split(',')]


def _groups(case):
    """Per sequence: (group, length, block list); per group the number of shared pages; pages in all.  Page 0 belongs to nobody, pages of a sequence lie
    anywhere.  The sequences that fill up a batch have length 0 and no pages."""
    sizes, prompts, bs = _ints(case['sizes']), _ints(case['prompts']), case['block']
    rng = random.Random(zlib.crc32(repr(sorted(case.items(), key=lambda kv: kv[0])).encode()))
    shared = [p // bs for p in prompts]
    rows = [(g, prompts[g] + rng.randint(1, case['answer'])) for g, n in enumerate(sizes) for _ in range(n)]
    need = sum(shared) + sum((n + bs - 1) // bs - shared[g] for g, n in rows)
    free = list(range(1, need + 1))
    rng.shuffle(free)
    take = iter(free)
    common = [[next(take) for _ in range(n)] for n in shared]
    seqs = [(g, n, common[g] + [next(take) for _ in range((n + bs - 1) // bs - shared[g])]) for g, n in rows]
    return seqs + [(-1, 0, [])] * case['fill'], shared, need + 1


def _cache(case, seed, blocks):
    shape = (blocks, case['block'], case['kv_heads'], case['dim'])
    B = sum(_ints(case['sizes'])) + case['fill']
    mk = lambda s, std, name: torch.empty(s, dtype=torch.bfloat16, device='cuda').normal_(0.0, std, generator=_gen(seed, name))  # noqa: E731
    # normed heads: scores of unit scale and a few keys that stand out
    return mk((B, case['heads'], case['dim']), 1.5, 'q'), mk(shape, 1.0, 'k'), mk(shape, 1.0, 'v')


def _pairs(case):
    """(source page, destination page, tokens) of a fork of every prompt, or of a compaction."""
    rng = random.Random(zlib.crc32(repr(sorted(case.items(), key=lambda kv: kv[0])).encode()))
    pages, bs = list(range(1, case['pages'])), case['block']
    rng.shuffle(pages)
    if case['mode'] == 'fork':
        out = []
        for _ in range(case['prompts']):
            src, filled = pages.pop(), rng.randint(1, bs - 1)
            out += [(src, pages.pop(), filled) for _ in range(case['samples'] - 1)]
        return out
    live = sorted({case['pages'] - 1, *pages[:case['prompts']]})
    holes = [p for p in range(1, len(live) + 1) if p not in set(live)]
    return [(s, d, bs) for s, d in zip(reversed(live), holes)]       # the last live page into the first hole: those that have a place in front stay


def _dtype(case):
    return torch.bfloat16 if case['type'] == 'bf16' else torch.float32


def _pools(case, seed):
    for n in range(case['layers']):
        for name, w in (('k', case['width']), ('v', case['value'])):
            yield torch.empty((case['pages'], case['block'], case['kv_heads'], w), dtype=_dtype(case), device='cuda').normal_(generator=_gen(seed, f'{name}{n}'))


def _tokens(case, seed):
    """Labels ``[rows, cols]``: a masked prompt, an answer, padding; now and then a row without an answer.  Log-probs of a model that knows most of its tokens."""
    B, S, g = case['rows'], case['cols'], _gen(seed, 'tokens')
    u = lambda: torch.rand(B, 1, device='cuda', generator=g)  # noqa: E731
    first, last = (u() * 0.4 * S).long(), (S * (0.5 + 0.5 * u())).long()
    last = torch.where(u() < 0.03, first, last)
    at = torch.arange(S, device='cuda')
    labels = torch.randint(0, 151936, (B, S), device='cuda', generator=g)
    labels = torch.where((at >= first) & (at < last), labels, torch.full_like(labels, -100))
    logps = -torch.empty(B, S, device='cuda').exponential_(2.0, generator=g)
    near = lambda std: torch.empty(B, S, device='cuda').normal_(0.0, std, generator=g)  # noqa: E731
    return labels, logps, near


def _policy(case, seed):
    labels, logps, near = _tokens(case, seed)
    B, S, g = case['rows'], case['cols'], _gen(seed, 'advantages')
    adv = torch.empty(B, S if case['advantage'] == 'token' else 1, device='cuda').normal_(generator=g)
    return {'labels': labels, 'logps': logps, 'advantages': adv if case['advantage'] == 'token' else adv[:, 0].contiguous(),
            'old': logps + near(0.15) if case['old'] else None, 'ref': logps + near(0.3) if case['beta'] else None,
            'entropies': torch.empty(B, S, device='cuda').exponential_(1.0, generator=g) if case['entropy'] else None}


def _prefer(case, seed):
    labels, logps, near = _tokens(case, seed)
    ref = logps + near(0.05) if case['reference'] != 'none' else None
    if case['reference'] == 'row':        # sums that were formed when the reference model ran
        ref = torch.where(labels != -100, ref, torch.zeros_like(ref)).double().sum(-1).float()
    return {'labels': labels, 'logps': logps, 'ref': ref}


def _policy_args(case):
    args = dict(ratio=case['ratio'], surrogate=case['surrogate'], reduce=case['reduce'], epsilon=0.2, epsilon_high=0.28, beta=case['beta'], entropy_coef=case['entropy'], tau=(1.0, 1.05))
    return dict(args, denominator=float(case['rows'] * 1024)) if case['reduce'] == 'sum' else args


def _prefer_args(case):
    return dict(form=case['form'], beta={'simpo': 2.5, 'orpo': 0.1}.get(case['form'], 0.1), gamma=0.5 if case['form'] == 'simpo' else 0.0, label_smoothing=case['smoothing'],
                nll_weight=1.0 if case['form'] == 'orpo' else case['nll'])


def prepare(case, seed):
    kind = case['kind']
    if kind == 'attend':
        seqs, shared, blocks = _groups(case)
        q, k, v = _cache(case, seed, blocks)
        table = torch.zeros(len(seqs), max(len(b) for _, _, b in seqs), dtype=torch.int32)
        for row, (_, _, b) in zip(table, seqs):
            row[:len(b)] = torch.tensor(b, dtype=torch.int32)
        sizes = _ints(case['sizes']) + [1] * case['fill']
        shared = shared + [0] * case['fill']
        state = {'kind': kind, 'q': q, 'k': k, 'v': v, 'table': table.cuda(), 'lens': torch.tensor([n for _, n, _ in seqs], dtype=torch.int32).cuda(), 'sizes': sizes, 'shared': shared}
        if own:
            from twinkle_b200 import ops
            state['plan'] = ops.shared_prefix(sizes, shared, case['block'], case['heads'], case['kv_heads'], device='cuda')
        return state
    if kind == 'copy':
        src, dst, tokens = map(list, zip(*_pairs(case)))
        return {'kind': kind, 'pools': list(_pools(case, seed)), 'src': src, 'dst': dst, 'tokens': tokens}
    if kind == 'policy':
        state = dict(_policy(case, seed), kind=kind, args=_policy_args(case))
        state['logps'].requires_grad_(own)
        if own and state['entropies'] is not None:
            state['entropies'].requires_grad_()
        return state
    state = dict(_prefer(case, seed), kind=kind, args=_prefer_args(case))
    state['logps'].requires_grad_(own)
    return state


# --------------------------------------------------------------- plain forms
def _attend(q, k, v, table, lens, sizes, shared):
    B, hq, D = q.shape
    bs, hkv = k.shape[1], k.shape[2]
    out, at = torch.zeros_like(q), 0
    for n, s in zip(sizes, shared):
        rows = slice(at, at + n)
        at += n
        qq = q[rows].float().view(n, hkv, hq // hkv, D) / math.sqrt(D)
        common = table[rows.start, :s].long()
        tail = table[rows, s:].long()
        kc, vc = k[common].float().view(-1, hkv, D), v[common].float().view(-1, hkv, D)
        kt, vt = k[tail].float().view(n, -1, hkv, D), v[tail].float().view(n, -1, hkv, D)
        at_c, at_t = torch.arange(kc.shape[0], device=q.device), kc.shape[0] + torch.arange(kt.shape[1], device=q.device)
        ln = lens[rows, None, None, None]
        scores = torch.cat([torch.einsum('nkgd,lkd->nkgl', qq, kc).masked_fill(at_c >= ln, float('-inf')),
                            torch.einsum('nkgd,nlkd->nkgl', qq, kt).masked_fill(at_t >= ln, float('-inf'))], -1)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - torch.where(top == float('-inf'), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        o = torch.einsum('nkgl,lkd->nkgd', p[..., :kc.shape[0]], vc) + torch.einsum('nkgl,nlkd->nkgd', p[..., kc.shape[0]:], vt)
        out[rows] = o.reshape(n, hq, D).to(out.dtype)
    return out


def _copy(pools, src, dst, tokens):
    bs = pools[0].shape[1]
    n = torch.tensor(tokens)
    pick = (torch.arange(bs) < n[:, None]).reshape(-1)
    rows = lambda x: (torch.tensor(x)[:, None] * bs + torch.arange(bs)).reshape(-1)[pick].cuda()  # noqa: E731
    s, d = rows(src), rows(dst)
    for p in pools:
        flat = p.view(-1, *p.shape[2:])
        flat[d] = flat[s]
    return pools


def _policy_loss(labels, logps, advantages, old, ref, entropies, ratio, surrogate, reduce, epsilon, epsilon_high, beta, entropy_coef, tau, denominator=None, wide=torch.float32):
    """Loss, figures and gradients by their formulas; ``wide``: the type of what is not a long sum, a difference of near numbers or next to a border."""
    f64 = torch.float64
    mask = labels != -100
    zero = torch.zeros((), dtype=f64, device=logps.device)
    masked = lambda x: torch.where(mask, x, torch.zeros_like(x))  # noqa: E731
    n = mask.sum(-1, keepdim=True).to(f64).clamp_min(1.0)
    total = mask.sum().to(f64)
    diff = masked(logps.to(f64) - (logps if old is None else old).to(f64))
    lr, inside = diff.clamp(-20.0, 20.0), (diff >= -20.0) & (diff <= 20.0)
    if ratio == 'sequence':
        lr = (lr.sum(-1, keepdim=True) / n).expand_as(lr)
    lo, hi = lr < math.log1p(-epsilon), lr > math.log1p(epsilon_high)
    adv = (advantages if advantages.dim() == 2 else advantages[:, None]).to(wide).expand_as(logps)
    r, r1 = torch.exp(lr.to(wide)), torch.expm1(lr.to(wide))
    if surrogate == 'clip':
        kept = torch.where(adv >= 0, ~hi, ~lo)
        bounded = torch.where(lo, torch.full_like(r, 1.0 - epsilon), torch.where(hi, torch.full_like(r, 1.0 + epsilon_high), r))
        f = -torch.minimum(r * adv, bounded * adv)
        df = torch.where(kept, -r * adv, torch.zeros_like(r))               # by the log ratio
        dlogp = torch.zeros_like(r)
    elif surrogate == 'soft':
        t = torch.where(adv > 0, torch.full_like(adv, tau[0]), torch.full_like(adv, tau[1]))
        gate = 1.0 / (1.0 + torch.exp(-t * r1))
        f, df, dlogp = -gate * 4.0 / t * adv, -4.0 * gate * (1.0 - gate) * r * adv, torch.zeros_like(r)
    else:
        weight = torch.where(lr > math.log1p(epsilon), torch.full_like(r, 1.0 + epsilon), r) * adv
        f, df, dlogp = -weight * logps.to(wide), torch.zeros_like(r), -weight
    if beta and ref is not None:
        d = masked(ref.to(f64) - logps.to(f64))
        f = f + (beta * (torch.expm1(d) - d)).to(wide)
        dlogp = dlogp - (beta * torch.expm1(d)).to(wide)
    if entropy_coef:
        f = f - entropy_coef * entropies.to(wide)
    if reduce == 'sequence':
        w = 1.0 / (n * logps.shape[0])
    else:
        w = (1.0 / (total.clamp_min(1.0) if reduce == 'token' else torch.full_like(total, denominator))).expand_as(n)
    loss = (masked(f).sum(-1, keepdim=True, dtype=f64) * w).sum()
    if ratio == 'sequence':
        df = (masked(df).sum(-1, keepdim=True, dtype=f64) / n).to(wide).expand_as(df)
    grad = masked((torch.where(inside, df, torch.zeros_like(df)) + dlogp) * w.to(wide))
    many = total.clamp_min(1.0)
    stats = torch.stack([masked(torch.expm1(lr) - lr).sum() / many, (lo & mask).sum() / many, (hi & mask).sum() / many, total + zero])
    out = {'loss': loss.to(wide), 'stats': stats.to(wide), 'logps': grad}
    if entropy_coef:
        out['entropies'] = masked((-entropy_coef * w).to(wide).expand_as(logps))
    return out


def _preference_loss(labels, logps, ref, form, beta, gamma, label_smoothing, nll_weight, wide=torch.float32):
    f64 = torch.float64
    mask = labels != -100
    n = mask.sum(-1).to(f64)
    sums = lambda x: torch.where(mask, x, torch.zeros_like(x)).sum(-1, dtype=f64)  # noqa: E731
    s = sums(logps)
    r = torch.zeros_like(s) if ref is None or form in ('simpo', 'orpo') else ref.to(f64) if ref.dim() == 1 else sums(ref)
    per = 1.0 / n.clamp_min(1.0) if form in ('simpo', 'orpo') else torch.ones_like(n)
    x = (s - r) * per
    c, j, pairs = x[0::2], x[1::2], s.numel() // 2
    soft = lambda z: torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))  # noqa: E731   log(1 + e^z)
    sig = lambda z: 1.0 / (1.0 + torch.exp(-z))  # noqa: E731
    z = beta * (c - j) - gamma
    if form in ('sigmoid', 'simpo'):
        f = soft(-z) * (1.0 - label_smoothing) + soft(z) * label_smoothing
        dz = -sig(-z) * (1.0 - label_smoothing) + sig(z) * label_smoothing
        dc, dj = beta * dz, -beta * dz
    elif form == 'hinge':
        f, dz = torch.clamp(1.0 - z, min=0.0), torch.where(z < 1.0, -torch.ones_like(z), torch.zeros_like(z))
        dc, dj = beta * dz, -beta * dz
    elif form == 'ipo':
        u = z - 1.0 / (2.0 * beta)
        f, dc, dj = u * u, 2.0 * beta * u, -2.0 * beta * u
    elif form == 'kto_pair':
        p, q = sig(beta * c), sig(beta * j)
        f, dc, dj = 1.0 - p + q, -beta * p * (1.0 - p), beta * q * (1.0 - q)
    else:
        most = math.log1p(-1e-6)          # of a probability that counts as certain
        rest = lambda a: torch.log(-torch.expm1(a.clamp(max=most)))  # noqa: E731
        odds = c - j - (rest(c) - rest(j))
        by = lambda a: torch.where(a <= most, 1.0 / -torch.expm1(a.clamp(max=most)), torch.ones_like(a))  # noqa: E731
        f, d = beta * soft(-odds), -beta * sig(-odds)
        dc, dj = d * by(c), -d * by(j)
    nc = n[0::2].sum().clamp_min(1.0)
    loss = f.mean() - nll_weight * s[0::2].sum() / nc
    coef = torch.stack([dc / pairs * per[0::2] - nll_weight / nc, dj / pairs * per[1::2]], -1).reshape(-1, 1)
    stats = torch.stack([beta * c.mean(), beta * j.mean(), beta * (c - j).mean(), (c > j).to(f64).mean(), s[0::2].mean(), s[1::2].mean()])
    grad = torch.where(mask, coef.to(wide), torch.zeros((), dtype=wide, device=mask.device))
    return {'loss': loss.to(wide), 'stats': stats.to(wide), 'logps': grad}


def run(state):
    kind = state['kind']
    if own:
        from twinkle_b200 import ops
        if kind == 'attend':
            return {'out': ops.paged_attention_shared(state['q'], state['k'], state['v'], state['table'], state['lens'], state['plan'])}
        if kind == 'copy':
            ops.cache_copy(state['pools'], state['src'], state['dst'], state['tokens'])
            return state['pools']
        if kind == 'policy':
            ent = state['entropies']
            loss, stats = ops.policy_loss(state['logps'], state['labels'], state['advantages'], state['old'], state['ref'], ent, **state['args'])
            grads = torch.autograd.grad(loss, [state['logps']] + ([] if ent is None else [ent]))
            return dict({'loss': loss.detach(), 'stats': stats}, **dict(zip(('logps', 'entropies'), grads)))
        loss, stats = ops.preference_loss(state['logps'], state['labels'], state['ref'], **state['args'])
        return {'loss': loss.detach(), 'stats': stats, 'logps': torch.autograd.grad(loss, state['logps'])[0]}
    if kind == 'attend':
        return {'out': _attend(state['q'], state['k'], state['v'], state['table'], state['lens'], state['sizes'], state['shared'])}
    if kind == 'copy':
        return _copy(state['pools'], state['src'], state['dst'], state['tokens'])
    if kind == 'policy':
        return _policy_loss(*(state[x] for x in ('labels', 'logps', 'advantages', 'old', 'ref', 'entropies')), **state['args'])
    return _preference_loss(state['labels'], state['logps'], state['ref'], **state['args'])


# ----------------------------------------------- what a pass cannot do without
def work(case):
    kind = case['kind']
    if kind == 'attend':
        seqs, shared, _ = _groups(case)
        hq, hkv, D = case['heads'], case['kv_heads'], case['dim']
        lens = [(g, n) for g, n, _ in seqs if g >= 0]
        rows = sum(n - shared[g] * case['block'] for g, n in lens) + sum(shared) * case['block']
        return {'bytes': 4 * rows * hkv * D + 4 * len(seqs) * hq * D, 'flops': 4 * hq * D * sum(n for _, n in lens)}
    if kind == 'copy':
        pairs = _pairs(case)
        token = case['layers'] * case['kv_heads'] * (case['width'] + case['value']) * _dtype(case).itemsize
        read = {}
        for s, _, n in pairs:
            read[s] = n
        return {'bytes': token * (sum(read.values()) + sum(n for _, _, n in pairs)), 'flops': 0}
    tokens = case['rows'] * case['cols']
    if kind == 'policy':
        per = 8 + 4 + 4 + 4 * case['old'] + 4 * (case['beta'] > 0) + 8 * (case['entropy'] > 0) + 4 * (case['advantage'] == 'token')
        return {'bytes': per * tokens, 'flops': 30 * tokens}
    return {'bytes': (8 + 4 + 4 + 4 * (case['reference'] == 'token')) * tokens, 'flops': 4 * tokens}


# ------------------------------------------------------------------ definitions
def exact(case, seed):
    kind = case['kind']
    if kind == 'attend':
        seqs, _, blocks = _groups(case)
        q, k, v = _cache(case, seed, blocks)
        hkv, D, bs = case['kv_heads'], case['dim'], case['block']
        out = torch.zeros(q.shape, dtype=torch.float64, device='cuda')
        for b, (_, n, pages) in enumerate(seqs):
            if n == 0:
                continue
            rows = torch.tensor(pages, device='cuda')
            for h in range(hkv):
                kk, vv = (x[rows, :, h].reshape(-1, D)[:n].double() for x in (k, v))
                heads = slice(h * (q.shape[1] // hkv), (h + 1) * (q.shape[1] // hkv))
                out[b, heads] = torch.softmax(q[b, heads].double() @ kk.t() * D ** -0.5, -1) @ vv
        return {'out': out}
    if kind == 'copy':
        where = torch.arange(case['pages'] * case['block'], device='cuda')          # the row that every row of a pool is taken from
        for s, d, n in _pairs(case):
            where[d * case['block']:d * case['block'] + n] = s * case['block'] + torch.arange(n, device='cuda')
        return [p.flatten(0, 1)[where].view(p.shape) for p in _pools(case, seed)]
    if kind == 'policy':
        return _exact_policy(case, seed)
    return _exact_prefer(case, seed)


def _exact_policy(case, seed):
    x, a = _policy(case, seed), _policy_args(case)
    if x['logps'].numel() > (1 << 23):
        return None
    f64 = lambda t: None if t is None else t.double()  # noqa: E731
    lp = x['logps'].double().requires_grad_()
    ent = x['entropies'].double().requires_grad_() if x['entropies'] is not None else None
    old, ref, adv = lp.detach() if x['old'] is None else f64(x['old']), f64(x['ref']), f64(x['advantages'])
    adv = (adv if adv.dim() == 2 else adv.unsqueeze(1)).expand(lp.shape)
    m = (x['labels'] != -100).double()
    count = m.sum(1, keepdim=True)
    log_ratio = torch.clamp(lp - old, -20, 20)
    if a['ratio'] == 'sequence':
        log_ratio = ((log_ratio * m).sum(1, keepdim=True) / count.clamp(min=1)).expand(lp.shape)
    rho = log_ratio.exp()
    if a['surrogate'] == 'clip':
        per = -torch.min(rho * adv, rho.clamp(1 - a['epsilon'], 1 + a['epsilon_high']) * adv)
    elif a['surrogate'] == 'soft':
        t = torch.where(adv > 0, a['tau'][0], a['tau'][1]).double()
        per = -torch.sigmoid(t * (rho - 1)) * 4 / t * adv
    else:
        per = -rho.clamp(max=1 + a['epsilon']).detach() * adv * lp
    if ref is not None:
        per = per + a['beta'] * ((ref - lp).exp() - (ref - lp) - 1)
    if ent is not None:
        per = per - a['entropy_coef'] * ent
    if a['reduce'] == 'sequence':
        loss = ((per * m).sum(1, keepdim=True) / count.clamp(min=1)).mean()
    else:
        loss = (per * m).sum() / (m.sum().clamp(min=1) if a['reduce'] == 'token' else a['denominator'])
    grads = torch.autograd.grad(loss, [lp] + ([] if ent is None else [ent]))
    with torch.no_grad():
        n = m.sum().clamp(min=1)
        stats = torch.stack([((rho - 1 - log_ratio) * m).sum() / n, ((rho < 1 - a['epsilon']) * m).sum() / n, ((rho > 1 + a['epsilon_high']) * m).sum() / n, m.sum()])
    return dict({'loss': loss.detach(), 'stats': stats}, **dict(zip(('logps', 'entropies'), grads)))


def _exact_prefer(case, seed):
    x, a = _prefer(case, seed), _prefer_args(case)
    if x['logps'].numel() > (1 << 23):
        return None
    lp = x['logps'].double().requires_grad_()
    m = (x['labels'] != -100).double()
    seq, count = (lp * m).sum(1), m.sum(1)
    form, beta, logsig = a['form'], a['beta'], torch.nn.functional.logsigmoid
    ref = torch.zeros_like(seq)
    if x['ref'] is not None and form not in ('simpo', 'orpo'):
        ref = x['ref'].double() if x['ref'].dim() == 1 else (x['ref'].double() * m).sum(1)
    level = seq / count.clamp(min=1) if form in ('simpo', 'orpo') else seq - ref
    c, r = level[0::2], level[1::2]
    z = beta * (c - r) - a['gamma']
    if form in ('sigmoid', 'simpo'):
        f = -logsig(z) * (1 - a['label_smoothing']) - logsig(-z) * a['label_smoothing']
    elif form == 'hinge':
        f = torch.relu(1 - z)
    elif form == 'ipo':
        f = (z - 1 / (2 * beta)) ** 2
    elif form == 'kto_pair':
        f = 1 - torch.sigmoid(beta * c) + torch.sigmoid(beta * r)
    else:
        f = -beta * logsig((c - r) - (torch.log1p(-c.exp().clamp(max=1 - 1e-6)) - torch.log1p(-r.exp().clamp(max=1 - 1e-6))))
    loss = f.mean() - a['nll_weight'] * seq[0::2].sum() / m[0::2].sum().clamp(min=1)
    grad, = torch.autograd.grad(loss, lp)
    stats = torch.stack([beta * c.mean(), beta * r.mean(), beta * (c - r).mean(), (c > r).double().mean(), seq[0::2].mean(), seq[1::2].mean()])
    return {'loss': loss.detach(), 'stats': stats.detach(), 'logps': grad}
