"""Operators of a policy step on the GPU against their 64-bit forms: decode over shared pages, copies of cache rows, policy and preference losses."""
import math

import pytest
import torch

from tests.policy_step_oracle import attention, batch, policy, preference
from tests.test_policy_step import BAD_COPIES, _tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def E():
    from twinkle_b200 import ops
    e = ops.ext()
    e.read_and_clear_error()
    yield e
    assert e.read_and_clear_error() == 0


# ------------------------------------------------------------- shared decode
def close(out, want, top):
    """Rounding to bf16 is within 2^-8 of the result.  A score is a sum of 128 products in fp32: within 128 · 2^-24 · |q| |k| / √128 ≈ 1.3e-4 for |q| = 1.5 √128, |k| = √128, so
    weights are within 2.6e-4 and, with their two bf16 parts (2^-16), a result within 2^-11 of the largest value.  These errors are independent: of the norm they are well below 2^-12."""
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    assert ((out - want).abs() <= 2**-8 * want.abs() + 2**-11 * top).all()
    assert (out - want).norm() <= (2**-8 + 2**-12) * want.norm()


SHAPES = [  # sizes, prompts, longest answer, page, query heads, key heads, width, sequences that fill the batch up
    ([1], [1], 0, 16, 8, 2, 128, 0), ([1], [16], 0, 16, 8, 2, 128, 0), ([2], [17], 3, 16, 8, 8, 64, 1), ([4], [509], 64, 16, 16, 8, 128, 0), ([8, 8], [128, 129], 40, 16, 32, 8, 128, 3),
    ([33, 1, 40], [700, 8, 127], 9, 8, 32, 8, 128, 0), ([5], [2000], 300, 24, 28, 4, 128, 0), ([130], [300], 20, 16, 8, 8, 64, 0), ([2, 3], [64, 40], 1, 64, 12, 2, 64, 0),
    ([3], [4100], 200, 128, 32, 4, 128, 1), ([2], [700], 5, 256, 8, 1, 128, 0), ([2], [300], 17, 16, 128, 1, 64, 0), ([3], [385], 2, 40, 16, 1, 128, 0), ([6, 2], [3, 5], 30, 16, 32, 8, 128, 0)]


@pytest.mark.parametrize('sizes,prompts,answers,bs,hq,hkv,D,fill', SHAPES)
def test_shared_decode(E, sizes, prompts, answers, bs, hq, hkv, D, fill):
    from twinkle_b200 import ops
    x, sizes, shared = batch(sizes, prompts, answers, bs, hq, hkv, D, device='cuda', fill=fill)
    q, k, v, table, lens = x
    # tokens that nobody holds are not read into any sum
    held = torch.zeros(k.shape[:2], dtype=torch.bool)
    for r, n in zip(table.cpu().tolist(), lens.tolist()):
        for t in range(n):
            held[r[t // bs], t % bs] = True
    k[~held.cuda()] = math.nan
    v[~held.cuda()] = math.inf
    plan = ops.shared_prefix(sizes, shared, bs, hq, hkv)
    before = E.launch_count()
    out = ops.paged_attention_shared(*x, plan)
    assert E.launch_count() - before == (3 if any(shared) else 1)
    close(out, *attention(*x))
    assert torch.equal(out, ops.paged_attention_shared(*x, plan))
    assert not out[len(out) - fill:].any()


@pytest.mark.parametrize('sizes,prompts,answers,bs,hq,hkv,D,fill', SHAPES)
def test_shared_decode_counts_every_token_once(E, sizes, prompts, answers, bs, hq, hkv, D, fill):
    """Equal scores: a result is a mean, here of the tokens' remainders by the width."""
    from twinkle_b200 import ops
    (q, k, v, table, lens), sizes, shared = batch(sizes, prompts, answers, bs, hq, hkv, D, device='cuda', fill=fill)
    q.zero_()
    v.zero_()
    for r, n in zip(table.tolist(), lens.tolist()):
        for t in range(n):
            v[r[t // bs], t % bs, :, t % D] = 1.0
    out = ops.paged_attention_shared(q, k, v, table, lens, ops.shared_prefix(sizes, shared, bs, hq, hkv)).double().cpu()
    for b, n in enumerate(lens.tolist()):
        want = torch.bincount(torch.arange(n) % D, minlength=D).double() / max(n, 1)
        assert ((out[b] - want).abs() <= (2**-8 + 2**-14) * want).all()


def test_shared_decode_of_sequences_shorter_than_their_prefix(E):
    from twinkle_b200 import ops
    x, sizes, shared = batch([6, 2], [200, 300], 20, 16, 16, 4, 128, device='cuda')
    for b, n in ((1, 0), (2, 5), (3, 191), (4, 192), (7, 17)):
        x[4][b] = n
    out = ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, 16, 16, 4))
    close(out, *attention(*x))
    assert not out[1].any()


def test_shared_decode_of_infinite_and_invalid_values(E):
    """An infinite value that a head weighs makes its dimension infinite, one that is not a number spoils its own dimension alone."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([4], [400], 10, 16, 16, 4, 128, device='cuda')
    q, k, v, table, lens = x
    p = table[0].tolist()
    v[p[3], 2, 0, 5], v[p[3], 3, 1, 6], v[p[20], 0, 2, 7] = math.inf, -math.inf, math.nan
    out = ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, 16, 16, 4))
    assert (out[:, 0:4, 5] == math.inf).all() and (out[:, 4:8, 6] == -math.inf).all() and out[:, 8:12, 7].isnan().all()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, 0:4, 5] = bad[:, 4:8, 6] = bad[:, 8:12, 7] = True
    assert torch.isfinite(out[~bad]).all()


def test_shared_decode_of_pages_outside_the_pool(E):
    """They count as zeros, nothing outside is read, and the error word says so."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([3], [64], 20, 16, 16, 4, 128, device='cuda')
    x[3][:, 1] = x[1].shape[0]
    x[3][1, -1] = -7
    plan = ops.shared_prefix(sizes, shared, 16, 16, 4)
    out = ops.paged_attention_shared(*x, plan)
    assert E.read_and_clear_error() != 0
    # a cache that has such pages, of zeros
    k, v = (torch.cat([t, torch.zeros_like(t[:1])]) for t in x[1:3])
    table = torch.where((x[3] < 0) | (x[3] >= x[1].shape[0]), torch.full_like(x[3], x[1].shape[0]), x[3])
    assert torch.equal(out, ops.paged_attention_shared(x[0], k, v, table, x[4], plan))


def test_shared_decode_far_into_a_pool(E):
    """Offsets beyond 2^31 elements."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([3], [200], 20, 16, 16, 8, 128, device='cuda')
    q, k, v, table, lens = x
    far = 140000 - k.shape[0]
    big = [torch.empty(140000, 16, 8, 128, dtype=torch.bfloat16, device='cuda') for _ in range(2)]
    for b, t in zip(big, (k, v)):
        b[far:].copy_(t)
    out = ops.paged_attention_shared(q, *big, table + far, lens, ops.shared_prefix(sizes, shared, 16, 16, 8))
    assert torch.equal(out, ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, 16, 16, 8)))


def test_shared_decode_in_graphs_and_on_a_stream(E):
    """Two captured calls and an eager one on another stream; a captured plan takes another plan's contents."""
    from twinkle_b200 import ops
    room = ops.prefix_items(6, 4)
    a, sa, ba = batch([4, 2], [333, 90], 30, 16, 16, 4, 128, seed=1, device='cuda')
    b, sb, bb = batch([1, 5], [700, 47], 30, 16, 16, 4, 128, seed=2, device='cuda')
    pa, pb = (ops.shared_prefix(s, n, 16, 16, 4, items=room) for s, n in ((sa, ba), (sb, bb)))
    want = [ops.paged_attention_shared(*x, p) for x, p in ((a, pa), (b, pb))]
    graphs, outs = [], []
    for x, p in ((a, pa), (b, pb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention_shared(*x, p))
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            other = ops.paged_attention_shared(*b, pb)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(other, want[1])
    # the same sequences in other groups: each on its own, with nothing shared
    again = ops.shared_prefix([1] * 6, [0] * 6, 16, 16, 4, items=room)
    pa.plan.copy_(again.plan)
    graphs[0].replay()
    close(outs[0], *attention(*a))


def test_shared_decode_of_other_types_reads_every_page(E):
    from twinkle_b200 import ops
    for dtype, bs, D in ((torch.float32, 16, 128), (torch.bfloat16, 12, 128), (torch.bfloat16, 16, 80)):
        x, sizes, shared = batch([3, 1], [50, 20], 9, bs, 8, 2, D, device='cuda', dtype=dtype)
        out = ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, bs, 8, 2))
        want, top = attention(*x)
        assert ((out.double().cpu() - want).abs() <= 2**-8 * want.abs() + 2**-11 * top).all()


def test_shared_decode_that_is_refused(E):
    from twinkle_b200 import ops
    x, sizes, shared = batch([3], [64], 20, 16, 16, 4, 128, device='cuda')
    with pytest.raises(ValueError):
        ops.paged_attention_shared(*x, ops.shared_prefix([2], shared, 16, 16, 4))
    with pytest.raises(ValueError):
        ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, 16, 32, 4))
    with pytest.raises(RuntimeError):       # the plan is elsewhere
        ops.paged_attention_shared(*x, ops.shared_prefix(sizes, shared, 16, 16, 4, device='cpu'))
    with pytest.raises(RuntimeError):
        ops.paged_attention_shared(*x[:4], x[4][:2], ops.shared_prefix(sizes, shared, 16, 16, 4))


# ------------------------------------------------------------------- copies
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize('widths', [(8, 8), (5, 3), (2, 128), (1, 1)])
@pytest.mark.parametrize('partly', [False, True])
def test_cache_copy(E, dtype, widths, partly):
    from twinkle_b200 import ops
    g = torch.Generator().manual_seed(1)
    pools = [torch.randint(0, 100, (50, 16) + widths[:1 + i % 2], generator=g).to(dtype).cuda() for i in range(5)]
    perm = torch.randperm(50, generator=g).tolist()
    src = perm[:20] + perm[:4]
    dst = perm[20:44]
    tokens = torch.randint(0, 17, (24, ), generator=g).tolist() if partly else None
    want = [p.cpu() for p in pools]
    ops.cache_copy(want, src, dst, tokens)
    ops.cache_copy(pools, src, dst, tokens)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(pools, want))


def test_cache_copy_of_many_pools_and_pairs(E):
    from twinkle_b200 import ops
    pools = [torch.randn(6000, 3, device='cuda') for _ in range(150)] + [None, torch.randn(6000, 40, device='cuda')]
    src, dst = list(range(0, 2500)), list(range(5999, 3499, -1))
    want = [p.clone() for p in pools if p is not None]
    for p in want:
        p[dst] = p[src]
    before = E.launch_count()
    ops.cache_copy(pools, src, dst)
    assert E.launch_count() - before == 4          # two of pools times two of pairs
    assert all(torch.equal(a, b) for a, b in zip([p for p in pools if p is not None], want))


def test_cache_copy_in_a_graph_and_on_a_stream(E):
    from twinkle_b200 import ops
    pool = torch.randn(8, 16, 64, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_copy([pool], [1], [2], [5])
    want = pool.clone()
    pool[1] = 7.0
    graph.replay()
    want[1] = 7.0
    want[2, :5] = 7.0
    assert torch.equal(pool, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_copy([pool], [1], [3])
    side.synchronize()
    assert (pool[3] == 7.0).all()


@pytest.mark.parametrize('src,dst,tokens', BAD_COPIES)
def test_cache_copies_that_are_refused(E, src, dst, tokens):
    from twinkle_b200 import ops
    pools = [torch.randn(6, 4, 3, device='cuda')]
    before = pools[0].clone()
    for bad in (pools, pools + [torch.randn(6, 4, 3, device='cuda').transpose(1, 2)], pools + [torch.randn(7, 4, 3, device='cuda')]):
        with pytest.raises(RuntimeError):
            ops.cache_copy(bad, src, dst, tokens)
    assert torch.equal(pools[0], before)


def test_cache_copy_far_into_a_pool(E):
    """Offsets beyond 2^32 bytes."""
    from twinkle_b200 import ops
    pool = torch.empty(150000, 16, 1024, dtype=torch.bfloat16, device='cuda')
    pool[3].normal_()
    pool[149998].normal_()
    ops.cache_copy([pool], [3, 149998], [149999, 4])
    assert torch.equal(pool[149999], pool[3]) and torch.equal(pool[4], pool[149998])


# ------------------------------------------------------------------- losses
def _policy_inputs(B, S, seed, masked='some'):
    labels, logps, near, g = _tokens(B, S, seed, masked)
    f = lambda t: t.float().cuda()  # noqa: E731
    x = dict(labels=labels.cuda(), logps=f(logps), old=f(near(0.3)), ref=f(near(0.3)), ent=torch.rand(B, S, generator=g).cuda(), adv=torch.randn(B, S, generator=g).cuda())
    x['old'][0, 0] = x['logps'][0, 0] + 30.0
    return x


def check_policy(x, adv, args, old=True, ref=True, ent=True):
    """Ratios are within 2^-21 and a token takes some five more roundings: within 2^-20 of its terms; the row's weight and its product with the token's derivative add 2^-23."""
    from twinkle_b200 import ops
    lp, en = x['logps'].detach().clone().requires_grad_(), x['ent'].detach().clone().requires_grad_()
    loss, stats = ops.policy_loss(lp, x['labels'], adv, x['old'] if old else None, x['ref'] if ref else None, en if ent else None, **args)
    grads = torch.autograd.grad(loss * 2.0, (lp, en) if ent else (lp, ))
    h = {n: t.detach().cpu() for n, t in x.items()}
    want = policy(h['logps'], h['labels'], adv.cpu(), h['old'] if old else None, h['ref'] if ref else None, h['ent'] if ent else None, **args)
    assert loss.dtype == torch.float32 and abs(float(loss.detach()) - want['loss']) <= 2**-20 * want['size'] + 2**-23 * abs(want['loss'])
    assert ((grads[0].double().cpu() / 2 - want['grad']).abs() <= 2**-19 * want['gsize']).all()
    if ent:
        assert ((grads[1].double().cpu() / 2 - want['gent']).abs() <= 2**-22 * want['gent'].abs()).all()
    for a, b in zip(stats.tolist(), want['stats']):
        assert abs(a - b) <= 2**-20 * abs(b)


@pytest.mark.parametrize('ratio', ['token', 'sequence'])
@pytest.mark.parametrize('surrogate', ['clip', 'soft', 'weight'])
@pytest.mark.parametrize('reduce', ['sequence', 'token', 'sum'])
@pytest.mark.parametrize('B,S', [(1, 1), (5, 37), (3, 2100)])
def test_policy_loss(E, ratio, surrogate, reduce, B, S):
    x = _policy_inputs(B, S, 3, 'some' if B > 1 else 'none')
    args = dict(ratio=ratio, surrogate=surrogate, reduce=reduce, epsilon=0.1, epsilon_high=0.3, beta=0.05, entropy_coef=0.02, tau=(1.0, 1.5), denominator=40.0)
    check_policy(x, x['adv'], args)


@pytest.mark.parametrize('case', ['row advantages', 'no old', 'bare', 'mask', 'all masked', 'rows apart', 'zero advantages', 'wide bound'])
def test_policy_loss_inputs(E, case):
    x = _policy_inputs(6, 300, 4)
    adv, args, has = x['adv'], dict(beta=0.1, entropy_coef=0.01), dict(old=True, ref=True, ent=True)
    if case == 'row advantages':
        adv = x['adv'][:, 7]                    # one number per row, S apart
    elif case == 'no old':
        has['old'] = False
    elif case == 'bare':
        args, has = {}, dict(old=True, ref=False, ent=False)
    elif case == 'mask':
        x['labels'] = x['labels'] != -100
    elif case == 'all masked':
        x['labels'].fill_(-100)
    elif case == 'rows apart':
        for n in x:
            wide = torch.zeros(6, 450, dtype=x[n].dtype, device='cuda')
            wide[:, 101:401] = x[n]
            x[n] = wide[:, 101:401]
        adv = x['adv']
    elif case == 'zero advantages':
        adv = torch.zeros_like(adv)
    else:
        args['epsilon'] = 1.5                   # no ratio is below a bound that is negative
    check_policy(x, adv, args, **has)


def test_policy_loss_ignores_masked_tokens(E):
    from twinkle_b200 import ops
    x = _policy_inputs(6, 300, 5)
    hide = x['labels'] == -100
    for ratio in ('token', 'sequence'):
        def run(y):
            lp = y['logps'].detach().clone().requires_grad_()
            loss, stats = ops.policy_loss(lp, y['labels'], y['adv'], y['old'], y['ref'], y['ent'], ratio=ratio, beta=0.1, entropy_coef=0.1)
            return loss.detach(), stats, torch.autograd.grad(loss, lp)[0]
        clean = run(x)
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
            y = {n: t if n == 'labels' else torch.where(hide, torch.full_like(t, bad), t) for n, t in x.items()}
            assert all(torch.equal(a, b) for a, b in zip(run(y), clean))
        assert not clean[2][hide].any()


@pytest.mark.parametrize('B,S', [(1, 70001), (700, 1), (300, 129), (64, 4095)])
@pytest.mark.parametrize('ratio', ['token', 'sequence'])
def test_policy_loss_of_many_tokens(E, B, S, ratio):
    """Against the plain form in 64 bits (checked against the definition on the CPU); terms are at most 2^3 here, so a token is within 2^-17 of its weight."""
    from twinkle_b200 import ops
    x = _policy_inputs(B, S, 6)
    args = dict(ratio=ratio, beta=0.1, entropy_coef=0.01, epsilon_high=0.28)
    lp, wide = x['logps'].detach().clone().requires_grad_(), x['logps'].double().requires_grad_()
    loss, stats = ops.policy_loss(lp, x['labels'], x['adv'], x['old'], x['ref'], x['ent'], **args)
    want, wstats = ops.ref.policy_loss(wide, x['labels'], x['adv'].double(), *(x[n].double() for n in ('old', 'ref', 'ent')), **args)
    grad, wgrad = torch.autograd.grad(loss, lp)[0], torch.autograd.grad(want, wide)[0]
    n = (x['labels'] != -100).sum(-1, keepdim=True).clamp_min(1)
    assert abs(float(loss.detach()) - float(want.detach())) <= 2**-17
    bound = 2**-17 / (n * B) if ratio == 'token' else 2**-17 / (n * B) * torch.ones_like(wgrad)
    assert ((grad.double() - wgrad).abs() <= bound).all()
    assert torch.allclose(stats.double(), wstats, rtol=2**-19, atol=1e-12)
    again = ops.policy_loss(lp, x['labels'], x['adv'], x['old'], x['ref'], x['ent'], **args)
    assert torch.equal(again[0], loss) and torch.equal(again[1], stats)


def test_policy_loss_at_the_bounds(E):
    """Log-probs of near numbers: the ratio's logarithm is formed in 64 bits and compared there."""
    from twinkle_b200 import ops
    old = torch.full((1, 4096), -1.0, device='cuda')
    lp = old + math.log(1.2) + torch.linspace(-1e-6, 1e-6, 4096, device='cuda')
    lp.requires_grad_()
    loss, stats = ops.policy_loss(lp, torch.ones(1, 4096, dtype=torch.bool, device='cuda'), torch.ones(1, device='cuda'), old)
    above = (lp.detach().double() - old.double()) > math.log1p(0.2)
    assert float(stats[2]) == float(above.float().mean())
    assert torch.equal(torch.autograd.grad(loss, lp)[0] == 0, above)


@pytest.mark.parametrize('form', ['sigmoid', 'hinge', 'ipo', 'kto_pair', 'simpo', 'orpo'])
@pytest.mark.parametrize('reference', ['token', 'row', 'none'])
@pytest.mark.parametrize('B,S', [(2, 1), (6, 41), (4, 5000)])
def test_preference_loss(E, form, reference, B, S):
    """All but the last rounding is in 64 bits: results are within 2^-23 of the definition's."""
    from twinkle_b200 import ops
    labels, logps, near, _ = _tokens(B, S, 7, 'some' if S > 1 else 'none')
    if form == 'orpo':
        labels[B // 2, :2] = 1                 # rows with an empty answer have no odds
    ref = near(0.01).float() if reference != 'none' else None
    if reference == 'row':
        ref = torch.where(labels != -100, ref, torch.zeros_like(ref)).sum(-1)
    args = dict(form=form, beta=0.3, gamma=0.2 if form == 'simpo' else 0.0, label_smoothing=0.1 if form == 'sigmoid' else 0.0, nll_weight=0.3)
    wide = logps.float().double().requires_grad_()
    want = preference(wide, labels, None if ref is None else ref.double(), **args)
    lp = logps.float().cuda().requires_grad_()
    loss, stats = ops.preference_loss(lp, labels.cuda(), None if ref is None else ref.cuda(), **args)
    grad, wgrad = torch.autograd.grad(loss * 0.5, lp)[0].double().cpu() * 2, torch.autograd.grad(want, wide)[0]
    assert abs(float(loss.detach()) - float(want.detach())) <= 2**-23 * abs(float(want.detach())) + 1e-12
    assert ((grad - wgrad).abs() <= 2**-22 * wgrad.abs() + 1e-30).all()
    plain = ops.ref.preference_loss(wide.detach(), labels, None if ref is None else ref.double(), **args)[1]
    assert torch.allclose(stats.double().cpu(), plain, rtol=2**-23, atol=1e-12)


def test_preference_loss_of_many_pairs(E):
    from twinkle_b200 import ops
    labels, logps, near, _ = _tokens(1200, 300, 8)
    lp, mask = logps.float().cuda(), labels.cuda() != -100
    ref = near(0.05).float().cuda()
    loss, stats = ops.preference_loss(lp, mask, ref)
    want, wstats = ops.ref.preference_loss(lp.double(), mask, ref.double())
    assert abs(float(loss) - float(want)) <= 2**-23 * float(want) and torch.allclose(stats.double(), wstats, rtol=2**-22)
    bad = torch.where(mask, lp, torch.full_like(lp, math.nan))
    assert torch.equal(ops.preference_loss(bad, mask, torch.where(mask, ref, torch.full_like(ref, math.inf)))[0], loss)


def test_losses_in_a_graph(E):
    """A captured step, forward and backward, replayed with other inputs; the eager graph of other leaves stays alive beside it."""
    from twinkle_b200 import ops
    x = _policy_inputs(4, 500, 9)
    eager_lp = x['logps'].detach().clone().requires_grad_()
    eager = ops.policy_loss(eager_lp, x['labels'], x['adv'], x['old'])[0], ops.preference_loss(eager_lp, x['labels'], x['ref'])[0]
    want = [torch.autograd.grad(l, eager_lp, retain_graph=True)[0] for l in eager]
    lp = torch.zeros_like(x['logps']).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step = lambda: [torch.autograd.grad(l, lp)[0] for l in (ops.policy_loss(lp, x['labels'], x['adv'], x['old'])[0], ops.preference_loss(lp, x['labels'], x['ref'])[0])]  # noqa: E731
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        lp.copy_(x['logps'])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('up', [math.inf, math.nan])
def test_masked_tokens_have_no_gradient_whatever_the_losses_is(E, up):
    from twinkle_b200 import ops
    x = _policy_inputs(4, 300, 16)
    lp, en = x['logps'].clone().requires_grad_(), x['ent'].clone().requires_grad_()
    losses = (ops.policy_loss(lp, x['labels'], x['adv'], x['old'], x['ref'], en, beta=0.1, entropy_coef=0.1)[0], ops.preference_loss(lp, x['labels'], x['ref'])[0])
    for loss in losses:
        for g in torch.autograd.grad(loss * up, (lp, en), allow_unused=True):
            assert g is None or (not g[x['labels'] == -100].any() and not torch.isfinite(g[x['labels'] != -100]).any())


def test_losses_have_no_second_derivative(E):
    from twinkle_b200 import ops
    x = _policy_inputs(4, 50, 11)
    lp = x['logps'].clone().requires_grad_()
    for loss in (ops.policy_loss(lp, x['labels'], x['adv'], x['old'])[0], ops.preference_loss(lp, x['labels'])[0]):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, lp, create_graph=True)


def test_policy_losses_out_of_the_kernels_range_keep_their_methods(E):
    from twinkle_b200.loss import GRPOLoss, SAPOLoss
    x = _policy_inputs(4, 50, 15)
    for loss in (SAPOLoss(tau_neg=-1.0), GRPOLoss(epsilon=-0.1)):
        before = E.launch_count()
        loss({'labels': x['labels']}, {'logps': x['logps']}, old_logps=x['old'], advantages=[1.0] * 4)
        assert E.launch_count() == before


def test_losses_keep_to_what_needs_a_gradient(E):
    from twinkle_b200 import ops
    x = _policy_inputs(4, 50, 10)
    with torch.no_grad():
        a = ops.policy_loss(x['logps'], x['labels'], x['adv'], x['old'], entropies=x['ent'], entropy_coef=0.1)[0]
    en = x['ent'].clone().requires_grad_()
    b = ops.policy_loss(x['logps'], x['labels'], x['adv'], x['old'], entropies=en, entropy_coef=0.1)[0]
    assert torch.equal(a, b.detach()) and not a.requires_grad
    assert torch.autograd.grad(b, en)[0].abs().sum() > 0
    # advantages that carry a gradient get it: the plain form takes over
    adv = x['adv'].clone().requires_grad_()
    c = ops.policy_loss(x['logps'], x['labels'], adv, x['old'])[0]
    assert torch.autograd.grad(c, adv)[0].abs().sum() > 0
    # log-probs in 16 bits
    half = x['logps'].bfloat16().requires_grad_()
    d = ops.policy_loss(half, x['labels'], x['adv'], x['old'])[0]
    assert torch.autograd.grad(d, half)[0].dtype == torch.bfloat16


# ------------------------------------------------------------- used together
def test_a_policy_step_end_to_end(E):
    """A group is sampled from a shared prompt on captured steps, its answers are scored and trained on: one run of all four operators."""
    from twinkle_b200 import ops
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.loss import DPOLoss, GRPOLoss
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.models.decoder import PackedBatch
    from twinkle_b200.sampler.engine import NativeEngine
    cfg = preset('qwen3-8b', num_hidden_layers=2, hidden_size=512, intermediate_size=1024, num_attention_heads=8, num_key_value_heads=2, vocab_size=1024)
    model = build_model(cfg, device='cuda', dtype=torch.bfloat16, seed=0)
    calls = {n: 0 for n in ('paged_attention_shared', 'cache_copy')}
    real = {n: getattr(ops, n) for n in calls}
    for n in calls:
        def counted(*a, _n=n, **k):
            calls[_n] += 1
            return real[_n](*a, **k)
        setattr(ops, n, counted)
    try:
        eng = NativeEngine(model, cfg, num_blocks=200, block_size=16, share_prompts=True)
        eng.share_from = 0
        prompts = [[(7 * i + 3) % 900 for i in range(300)], [(3 * i + 1) % 900 for i in range(64)]]
        res = eng.generate(prompts, [SamplingParams(max_tokens=20, temperature=1.0, num_samples=4) for _ in prompts])
    finally:
        for n, f in real.items():
            setattr(ops, n, f)
    assert calls['cache_copy'] == 1 and calls['paged_attention_shared'] > 0 and any(k[2] for k in eng._graphs)
    # the log-prob of every sampled token, from a forward over the whole answer
    rows = [(p, s) for p, r in zip(prompts, res) for s in r.sequences]
    assert len(rows) == 8 and sorted(eng.cache.free) == list(range(1, 200))
    S = max(len(p) + len(s.tokens) for p, s in rows)
    labels, logps, old = torch.full((8, S), -100), [], torch.zeros(8, S)
    hidden = []
    for b, (p, s) in enumerate(rows):
        toks, n = p + s.tokens, len(p)
        batch_ = PackedBatch(torch.tensor(toks, device='cuda'), torch.arange(len(toks), device='cuda'), torch.tensor([0, len(toks)], dtype=torch.int32, device='cuda'), len(toks))
        with torch.no_grad():
            hidden.append(model(batch_))
        labels[b, n - 1:len(toks) - 1] = torch.tensor(s.tokens)
        old[b, n - 1:len(toks) - 1] = torch.tensor(s.logprobs)
    x = torch.zeros(8, S, 512, dtype=torch.bfloat16, device='cuda')
    for b, h in enumerate(hidden):
        x[b, :h.shape[0]] = h
    x.requires_grad_()
    flat = labels.clamp_min(0).reshape(-1).cuda()
    logps = ops.fused_linear_logprob(x.reshape(8 * S, 512), model.head_weight().detach(), flat)[0].view(8, S)
    mask = labels != -100
    assert (logps.detach().cpu() - old)[mask].abs().max() < 0.05          # bf16 activations of two routes through the model
    losses = [GRPOLoss(epsilon=0.2, beta=0.04)({'labels': labels}, {'logps': logps}, old_logps=old, ref_logps=old, advantages=[1.0, -1.0, 0.5, -0.5] * 2)['loss'],
              DPOLoss(beta=0.1)({'labels': labels}, {'logps': logps}, ref_logps=old)['loss']]
    for loss in losses:
        g, = torch.autograd.grad(loss, x, retain_graph=True)
        assert torch.isfinite(g).all() and g[mask.cuda()].abs().sum() > 0 and not g[~mask.cuda()].any()


@pytest.mark.parametrize('stack', ['tiny-dense', 'tiny-hybrid', 'tiny-deepseek', 'pomelix', 'moronex', 'puzonex'])
def test_groups_share_their_prompt(E, stack, tmp_path):
    """Greedy answers of a group in fp32 are those of separate sequences; in bf16 a captured and an eager step agree."""
    from tests.test_policy_step import _engine, run_group
    runs = [run_group(_engine(stack, tmp_path, ('cuda', 'float32'), share=s)) for s in (False, True)]
    for a, b in zip(*runs):
        for x, y in zip(a.sequences, b.sequences):
            assert x.tokens == y.tokens and x.logprobs == pytest.approx(y.logprobs, abs=1e-3)
    got = []
    for graphs in (True, False):
        e = _engine(stack, tmp_path, ('cuda', 'bfloat16'), share=True)
        e.use_cuda_graphs = graphs
        got.append(run_group(e))
        assert sorted(e.cache.free) == list(range(1, e.cache.num_blocks)) and not e.cache.sharers
    for a, b in zip(*got):
        for x, y in zip(a.sequences, b.sequences):
            assert x.tokens == y.tokens and x.logprobs == pytest.approx(y.logprobs, abs=1e-3)


def test_a_group_that_shrinks_and_is_compacted(E):
    """Steps of a group on captured graphs, with fewer members from step to step and the cache compacted in between, against separate sequences."""
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.sampler.engine import NativeEngine, _Seq
    cfg = preset('qwen3-8b', num_hidden_layers=2, hidden_size=512, intermediate_size=1024, num_attention_heads=8, num_key_value_heads=2, vocab_size=1024)
    model = build_model(cfg, device='cuda', dtype=torch.bfloat16, seed=0)
    prompt = [(7 * i + 3) % 900 for i in range(211)]
    steps = {}
    for share in (False, True):
        eng = NativeEngine(model, cfg, num_blocks=160, block_size=16, max_batch=8, share_prompts=share)
        eng.share_from = 0
        seqs = [_Seq(0, list(prompt), SamplingParams(max_tokens=8)) for _ in range(6)] + [_Seq(1, prompt[:40], SamplingParams(max_tokens=8))]
        if share:
            eng.prefill([seqs[0], seqs[6]])
            eng.fork(seqs[0], seqs[1:6])
        else:
            eng.prefill(seqs)
        steps[share] = []
        for n in range(5):
            for i, s in enumerate(seqs):
                s.tokens.append((37 * n + s.request + 11 * len(seqs)) % 900)
            steps[share].append(eng.decode_step(seqs, torch.tensor([s.tokens[-1] for s in seqs], device='cuda')).clone())
            if n in (1, 2):
                eng.release([seqs.pop(0)])
            if n == 2:
                eng.compact(seqs, 100)
    for a, b in zip(steps[False], steps[True]):
        assert (a - b).norm() / a.norm() < 2e-2
    assert E.read_and_clear_error() == 0


@pytest.mark.parametrize('name,kwargs', [('GRPOLoss', dict(epsilon=0.2, epsilon_high=0.3, beta=0.05)), ('GRPOLoss', dict(entropy_coef=0.01)), ('GSPOLoss', dict(epsilon=0.01)),
                                         ('SAPOLoss', dict(tau_neg=1.5)), ('CISPOLoss', dict(epsilon=0.1)), ('BNPOLoss', {}), ('DRGRPOLoss', dict(max_completion_length=64))])
@pytest.mark.parametrize('form', ['rows', 'list', 'ragged', 'tokens', 'one'])
def test_policy_loss_classes(E, name, kwargs, form):
    """The classes on the GPU against their methods on the CPU, however the advantages come."""
    from twinkle_b200 import loss as L
    x = _policy_inputs(6, 80, 12)
    labels = x['labels'].cpu()
    adv = {'rows': x['adv'][:, 0], 'list': x['adv'][:, 0].tolist(), 'ragged': [r[m].tolist() for r, m in zip(x['adv'].cpu(), labels != -100)], 'tokens': x['adv'], 'one': 0.7}[form]
    if form == 'ragged':
        adv = [r or [0.0] for r in adv]
    got = []
    for device in ('cuda', 'cpu'):
        lp = x['logps'].detach().to(device).requires_grad_()
        before = E.launch_count()
        out = getattr(L, name)(**kwargs)({'labels': labels}, {'logps': lp, 'entropies': x['ent'].to(device)}, old_logps=x['old'].to(device), ref_logps=x['ref'].to(device), advantages=adv)['loss']
        assert (E.launch_count() > before) == (device == 'cuda')
        got.append((out.detach().cpu(), torch.autograd.grad(out, lp)[0].cpu()))
    (a, ga), (b, gb) = got
    # the methods work in fp32 throughout: 480 terms of up to 2^3 of either sign
    assert abs(float(a - b)) <= 2**-17 * max(1.0, abs(float(b))) and (ga - gb).abs().max() <= 2**-17 * gb.abs().max()


def test_policy_losses_of_other_rules_keep_their_methods(E):
    from twinkle_b200.loss import GRPOLoss

    class Mine(GRPOLoss):
        def _surrogate(self, ratio, adv, logps):
            return -ratio * adv * 3.0

    x = _policy_inputs(4, 20, 13)
    before = E.launch_count()
    got = Mine()({'labels': x['labels']}, {'logps': x['logps']}, old_logps=x['logps'], advantages=[1.0] * 4)['loss']
    assert E.launch_count() == before and abs(float(got) + 3.0 * float(((x['labels'] != -100).any(-1)).float().mean())) < 1e-5


@pytest.mark.parametrize('name,kwargs', [('DPOLoss', dict(loss_type=t)) for t in ('sigmoid', 'hinge', 'ipo', 'kto_pair')] +
                         [('DPOLoss', dict(label_smoothing=0.1, sft_weight=0.3)), ('DPOLoss', dict(reference_free=True)), ('SimPOLoss', {}), ('CPOLoss', {}), ('ORPOLoss', {})])
@pytest.mark.parametrize('form', ['tokens', 'short', 'long', 'rows', 'pairs'])
def test_preference_loss_classes(E, name, kwargs, form):
    from twinkle_b200 import loss as L
    x = _policy_inputs(6, 40, 14)
    x['labels'][3, 1] = 5                     # no row without an answer
    labels, ref = x['labels'].cpu(), x['ref'].cpu()
    seq = torch.where(labels != -100, ref, torch.zeros_like(ref)).sum(-1)
    extra = {'tokens': dict(ref_logps=ref), 'short': dict(ref_outputs={'logps': ref[:, :30]}), 'long': dict(ref_logps=torch.cat([ref, ref], 1)), 'rows': dict(ref_logps=seq),
             'pairs': dict(ref_chosen_logps=seq[0::2], ref_rejected_logps=seq[1::2])}[form]
    if kwargs.get('reference_free') and form == 'tokens':
        extra = {}
    got, stats = [], []
    for device in ('cuda', 'cpu'):
        lp = x['logps'].detach().to(device).requires_grad_()
        before = E.launch_count()
        obj = getattr(L, name)(**kwargs)
        out = obj({'labels': labels}, {'logps': lp}, **extra)['loss']
        assert (E.launch_count() > before) == (device == 'cuda')
        got.append((out.detach().cpu(), torch.autograd.grad(out, lp)[0].cpu()))
        stats.append(getattr(obj, 'last_stats', {}))
    (a, ga), (b, gb) = got
    assert abs(float(a - b)) <= 2**-16 * max(1.0, abs(float(b))) and (ga - gb).abs().max() <= 2**-15 * gb.abs().max()
    assert stats[0].keys() == stats[1].keys() and all(stats[0][k] == pytest.approx(stats[1][k], rel=1e-4, abs=1e-4) for k in stats[0])
