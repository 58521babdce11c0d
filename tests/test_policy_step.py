"""Operators of a policy step on the CPU: plans of shared prefixes, copies of cache rows, the losses' plain forms and what the entry points refuse."""
import math
import random

import pytest
import torch

from tests.policy_step_oracle import attention, batch, policy, preference
from twinkle_b200 import ops


def test_pieces_of_shared_prefixes_cover_every_block_once():
    rng = random.Random(1)
    for _ in range(300):
        sizes = [rng.choice([1, 2, 8, 13, 40, rng.randint(1, 130)]) for _ in range(rng.randint(1, 12))]
        bs, G, hkv = rng.choice([8, 16, 24, 64, 128]), rng.choice([1, 2, 4, 5, 7, 8, 128]), rng.choice([1, 2, 4, 8])
        blocks = [rng.choice([0, 1, 3, rng.randint(0, 2000)]) for _ in sizes]
        items, lines = ops._prefix_items(sizes, blocks, bs, G, hkv, 148)
        assert len(items) <= ops.prefix_items(sum(sizes), hkv, 'cpu')
        group = [g for g, n in enumerate(sizes) for _ in range(n)]
        first = [sum(sizes[:g]) for g in group]
        for b, (tokens, slot, slots, row) in enumerate(lines):
            g = group[b]
            if not blocks[g]:
                assert slots == 0
                continue
            assert tokens == blocks[g] * bs and slots > 0
            at = 0
            for s in range(slot, slot + slots):
                row0, n, lo, count, t, mine, _, _ = items[s]
                assert mine == s and t == tokens and first[b] <= row0 <= b < row0 + n <= first[b] + sizes[g] and row == (b - row0) * G and n * G <= 128
                assert lo == at and count > 0
                at += count
            assert at == (tokens + 127) // 128


def test_plan_has_room_for_another():
    p = ops.shared_prefix([3, 1], [4, 0], 16, 8, 4, device='cpu', items=40)
    assert p.items == p.slots == 40 and p.plan.numel() == 40 * 8 + 4 * 4 and p.sequences == 4
    assert ops.shared_prefix([2], [0], 16, 8, 4, device='cpu').items == 0


@pytest.mark.parametrize('args', [([0], [1], 16, 8, 4), ([1, 2], [1], 16, 8, 4), ([1], [-1], 16, 8, 4), ([1], [1], 0, 8, 4), ([1], [1], 16, 8, 3), ([1], [1], 16, 258, 2)])
def test_plans_that_are_refused(args):
    with pytest.raises(ValueError):
        ops.shared_prefix(*args, device='cpu')


def test_shared_decode_on_the_cpu_is_attention_over_the_whole_table():
    x, sizes, shared = batch([3, 2], [37, 16], 9, 16, 4, 2, 32, dtype=torch.float32, fill=1)
    plan = ops.shared_prefix(sizes, shared, 16, 4, 2, device='cpu')
    got = ops.paged_attention_shared(*x, plan)
    want, _ = attention(*x)
    assert (got.double() - want).abs().max() < 1e-5 and not got[-1].any()
    with pytest.raises(ValueError):       # a plan of other sequences
        ops.paged_attention_shared(x[0][:2], x[1], x[2], x[3][:2], x[4][:2], plan)


# ------------------------------------------------------------------- copies
def test_cache_copy_copies_rows_of_all_pools():
    pools = [torch.randn(6, 4, 3), torch.randn(6, 4, 2, 5), None]
    before = [p.clone() for p in pools[:2]]
    ops.cache_copy(pools, [1, 1, 4], [0, 5, 2])
    for p, b in zip(pools, before):
        assert torch.equal(p[[0, 5, 2]], b[[1, 1, 4]]) and torch.equal(p[[1, 3, 4]], b[[1, 3, 4]])
    ops.cache_copy(pools, [3, 4], [0, 5], tokens=[2, 0])
    assert torch.equal(pools[0][0, :2], before[0][3, :2]) and torch.equal(pools[0][0, 2:], before[0][1, 2:]) and torch.equal(pools[0][5], before[0][1])
    ops.cache_copy(pools, [], [])


BAD_COPIES = [([0], [6], None), ([-1], [0], None), ([0, 1], [2, 2], None), ([0, 1], [1, 2], None), ([0], [0], None), ([0], [1], [5]), ([0], [1], [-1])]


@pytest.mark.parametrize('src,dst,tokens', BAD_COPIES)
def test_cache_copies_that_are_refused(src, dst, tokens):
    pools = [torch.randn(6, 4, 3)]
    before = pools[0].clone()
    with pytest.raises(RuntimeError):
        ops.cache_copy(pools, src, dst, tokens)
    assert torch.equal(pools[0], before)
    with pytest.raises(ValueError):
        ops.cache_copy(pools, [0, 1], [2])
    for few in ([1], []):
        with pytest.raises(ValueError):
            ops.cache_copy(pools, [0, 1], [2, 3], few)


# ------------------------------------------------------------------- losses
def _tokens(B, S, seed, masked='some'):
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(0, 100, (B, S), generator=g)
    if masked == 'some':
        labels[torch.rand(B, S, generator=g) < 0.4] = -100
        labels[B // 2] = -100                 # a row without tokens
    logps = -torch.empty(B, S, dtype=torch.float64).exponential_(1.0, generator=g)
    near = lambda s: logps + s * torch.randn(B, S, dtype=torch.float64, generator=g)  # noqa: E731
    return labels, logps, near, g


@pytest.mark.parametrize('ratio', ['token', 'sequence'])
@pytest.mark.parametrize('surrogate', ['clip', 'soft', 'weight'])
@pytest.mark.parametrize('reduce', ['sequence', 'token', 'sum'])
def test_policy_loss_plain_form(ratio, surrogate, reduce):
    labels, logps, near, g = _tokens(5, 7, 3)
    adv, old, ref, ent = torch.randn(5, 7, dtype=torch.float64, generator=g), near(0.3), near(0.3), torch.rand(5, 7, dtype=torch.float64, generator=g)
    old[0, 0] = logps[0, 0] + 30.0            # beyond the clamp
    args = dict(ratio=ratio, surrogate=surrogate, reduce=reduce, epsilon=0.1, epsilon_high=0.3, beta=0.05, entropy_coef=0.02, tau=(1.0, 1.5), denominator=40.0)
    lp, e = logps.clone().requires_grad_(), ent.clone().requires_grad_()
    loss, stats = ops.policy_loss(lp, labels, adv, old, ref, e, **args)
    grads = torch.autograd.grad(loss, (lp, e))
    want = policy(logps, labels, adv, old, ref, ent, **args)
    assert abs(float(loss.detach()) - want['loss']) < 1e-12 and (grads[0] - want['grad']).abs().max() < 1e-12 and (grads[1] - want['gent']).abs().max() < 1e-12
    assert torch.allclose(stats, torch.tensor(want['stats'], dtype=torch.float64), atol=1e-12)
    # a difference of the loss (the gate of the weighted form is held fixed: no difference shows that)
    if surrogate != 'weight':
        t = int((labels[1] != -100).nonzero()[0])
        up, down = logps.clone(), logps.clone()
        up[1, t] += 1e-6
        down[1, t] -= 1e-6
        diff = (ops.policy_loss(up, labels, adv, old, ref, ent, **args)[0] - ops.policy_loss(down, labels, adv, old, ref, ent, **args)[0]) / 2e-6
        assert abs(float(diff) - float(want['grad'][1, t])) < 1e-7


@pytest.mark.parametrize('form', ['sigmoid', 'hinge', 'ipo', 'kto_pair', 'simpo', 'orpo'])
@pytest.mark.parametrize('reference', ['token', 'row', 'none'])
def test_preference_loss_plain_form(form, reference):
    labels, logps, near, _ = _tokens(6, 5, 4)
    labels[3] = torch.arange(5)
    ref = near(0.5) if reference != 'none' else None
    if reference == 'row':
        ref = torch.where(labels != -100, ref, torch.zeros_like(ref)).sum(-1)
    args = dict(form=form, beta=0.7, gamma=0.2 if form == 'simpo' else 0.0, label_smoothing=0.1 if form == 'sigmoid' else 0.0, nll_weight=0.3)
    labels[2] = torch.arange(5)               # rows with an empty answer have no odds
    a, b = logps.clone().requires_grad_(), logps.clone().requires_grad_()
    loss, stats = ops.preference_loss(a, labels, ref, **args)
    want = preference(b, labels, ref, **args)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-12
    assert (torch.autograd.grad(loss, a)[0] - torch.autograd.grad(want, b)[0]).abs().max() < 1e-12
    assert stats.shape == (6, ) and torch.isfinite(stats).all()


def test_masked_tokens_do_not_reach_a_loss():
    labels, logps, near, g = _tokens(4, 6, 5)
    hide = labels == -100
    old, adv = near(0.2), torch.randn(4, 6, dtype=torch.float64, generator=g)
    clean = ops.policy_loss(logps, labels, adv, old)[0], ops.preference_loss(logps, labels, old)[0]
    for bad in (math.nan, math.inf, -math.inf):
        x = [torch.where(hide, torch.full_like(t, bad), t) for t in (logps, old, adv)]
        lp = x[0].requires_grad_()
        got = ops.policy_loss(lp, labels, x[2], x[1])[0], ops.preference_loss(lp, labels, x[1])[0]
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
        assert all(torch.isfinite(torch.autograd.grad(y, lp, retain_graph=True)[0]).all() for y in got)


def test_losses_that_are_refused():
    lp, y, a = torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.int64), torch.randn(4)
    for bad in (dict(ratio='row'), dict(surrogate='none'), dict(reduce='mean'), dict(epsilon=-0.1), dict(denominator=0.0), dict(tau=(0.0, 1.0)), dict(entropy_coef=0.1),
                dict(old_logps=torch.zeros(4)), dict(ref_logps=torch.zeros(4, 2), beta=0.1)):
        with pytest.raises(ValueError):
            ops.policy_loss(lp, y, a, **bad)
    with pytest.raises(ValueError):
        ops.policy_loss(lp, y[:, :2], a)
    with pytest.raises(ValueError):
        ops.policy_loss(lp, y, a[:3])
    with pytest.raises(ValueError):
        ops.policy_loss(lp[0], y[0], a)
    for bad in (dict(form='none'), dict(form='ipo', beta=0.0), dict(ref_logps=torch.zeros(3))):
        with pytest.raises(ValueError):
            ops.preference_loss(lp, y, **bad)
    with pytest.raises(ValueError):
        ops.preference_loss(lp[:3], y[:3])


# -------------------------------------------------------- sampling of groups
def _engine(stack, tmp_path, where=('cpu', 'float32'), share=False, block_size=16, num_blocks=96):
    import importlib
    from twinkle_b200.sampler import TorchSampler
    args = {'num_blocks': num_blocks, 'block_size': block_size, 'max_batch': 16, 'share_prompts': share}
    path = stack
    if not stack.startswith('tiny'):       # a listed-layer stack
        oracle, name = importlib.import_module(f'tests.{stack}_oracle'), 'mixed'
        path = str(tmp_path / stack)
        if not (tmp_path / stack).exists():
            (tmp_path / stack).mkdir()
            oracle.write_checkpoint(path, oracle.CONFIGS[name], oracle.random_weights(oracle.CONFIGS[name], 0))
    engine = TorchSampler(model_id=path, device=where[0], enable_lora=False, dtype=where[1], engine_args=args).engine
    engine.share_from = 0            # however little there is to share
    return engine


def run_group(engine, samples=3, max_tokens=9):
    """Prompts that end inside and at the end of a page, one twice; a request that is only scored."""
    from twinkle_b200.data_format import SamplingParams
    prompts = [[(7 * i + 3) % 90 for i in range(n)] for n in (37, 32, 5, 37)] + [[(5 * i + 1) % 90 for i in range(20)]]
    params = [SamplingParams(max_tokens=max_tokens, temperature=0.0, num_samples=samples) for _ in prompts]
    params[2].num_samples = 1
    params[4] = SamplingParams(max_tokens=0, prompt_logprobs=0, num_samples=2)
    return engine.generate(prompts, params)


STACKS = ['tiny-dense', 'tiny-hybrid', 'tiny-deepseek', 'tiny-gpt-oss', 'pomelix', 'moronex', 'nilepel', 'puzonex']


@pytest.mark.parametrize('stack', STACKS)
def test_groups_share_their_prompt(stack, tmp_path):
    free, runs = {}, {}
    for share in (False, True):
        e = _engine(stack, tmp_path, share=share)
        fed = []
        prefill = e.prefill
        e.prefill = lambda seqs: (fed.extend(len(s.prompt) for s in seqs), prefill(seqs))[1]
        runs[share] = run_group(e)
        free[share] = (sorted(e.cache.free), sorted(e.cache.free_slots), e.cache.sharers)
        assert sorted(fed) == (sorted([5, 32, 37, 20]) if share else sorted([37] * 6 + [32] * 3 + [5] + [20] * 2))
    assert free[True] == free[False] and free[True][2] == {}
    for a, b in zip(runs[True], runs[False]):
        assert len(a.sequences) == len(b.sequences)
        assert a.prompt_logprobs is None if b.prompt_logprobs is None else a.prompt_logprobs[1:] == pytest.approx(b.prompt_logprobs[1:], abs=1e-4)
        for x, y in zip(a.sequences, b.sequences):
            assert x.tokens == y.tokens and x.logprobs == pytest.approx(y.logprobs, abs=1e-4)


def test_forks_own_what_they_write():
    from twinkle_b200.models import preset
    from twinkle_b200.sampler.engine import PagedKVCache
    c = PagedKVCache(preset('tiny-dense'), 20, 4, torch.device('cpu'), torch.float32)
    first = c.allocate(4)
    lists, copies = c.fork(first, 10, [4, 3, 1])
    assert [l[:2] for l in lists] == [first[:2]] * 3 and [len(l) for l in lists] == [4, 3, 3]
    assert copies == [(first[2], l[2], 2) for l in lists] and len({b for l in lists for b in l[2:]} | set(first)) == 8
    for k in c.k + c.v:
        k.copy_(torch.randn(k.shape))
    before = [k.clone() for k in c.k + c.v]
    c.copy(copies)
    for k, b in zip(c.k + c.v, before):
        for l in lists:
            assert torch.equal(k[l[2], :2], b[first[2], :2]) and torch.equal(k[l[2], 2:], b[l[2], 2:])
    c.release(first)
    assert not set(first[:2]) & set(c.free) and set(first[2:]) <= set(c.free)
    for l in lists:
        c.release(l)
    assert sorted(c.free) == list(range(1, 20)) and not c.sharers
    whole, copies = c.fork(c.allocate(2), 8, [3])
    assert copies == [] and len(whole[0]) == 3
    with pytest.raises(RuntimeError):
        c.fork(whole[0], 12, [40])


def test_sequences_of_a_group_compare_and_print():
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.sampler.engine import _Seq
    a, b = (_Seq(0, [1, 2], SamplingParams()) for _ in range(2))
    a.origin, b.origin = a, a
    assert a == b and 'prompt' in repr(a)


def test_compaction_keeps_what_is_alive():
    from twinkle_b200.models import preset
    from twinkle_b200.sampler.engine import PagedKVCache
    c = PagedKVCache(preset('tiny-dense'), 24, 4, torch.device('cpu'), torch.float32)
    for k in c.k + c.v:
        k.copy_(torch.randn(k.shape))
    a, b, gone = c.allocate(3), c.allocate(4), c.allocate(9)
    d = c.allocate(3)
    (e, ), _ = c.fork(b, 8, [4])
    c.release(gone)
    lists = [a, b, d, e]
    rows = [[k[l].clone() for k in c.k + c.v] for l in lists]
    with pytest.raises(RuntimeError):        # a list is missing
        c.compact(lists[:3])
    with pytest.raises(RuntimeError):
        c.compact(lists, 12)
    c.compact(lists, 14)
    assert c.k[0].shape[0] == 14 and sorted({x for l in lists for x in l}) == list(range(1, 13)) and c.free == [13] and e[:2] == b[:2]
    assert all(torch.equal(k[l], r) for l, held in zip(lists, rows) for k, r in zip(c.k + c.v, held))
    c.compact(lists, 30)
    for l in lists:
        c.release(l)
    assert sorted(c.free) == list(range(1, 30)) and not c.sharers


def test_compaction_between_steps():
    """Sequences go on from a cache that was compacted and cut while they were alive."""
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.sampler.engine import NativeEngine, _Seq
    cfg = preset('tiny-dense')
    model = build_model(cfg, device='cpu', dtype=torch.float32, seed=0)
    out = []
    for compact in (False, True):
        eng = NativeEngine(model, cfg, num_blocks=64, block_size=4, max_batch=8, share_prompts=True)
        seqs = [_Seq(0, [3, 4, 5, 6, 7, 8], SamplingParams(max_tokens=4)) for _ in range(4)]
        eng.prefill(seqs[:1])
        eng.fork(seqs[0], seqs[1:])
        lone = _Seq(1, [9] * 10, SamplingParams(max_tokens=4))
        eng.prefill([lone])
        for n in range(3):
            for i, s in enumerate(seqs + [lone]):
                s.tokens.append(10 * n + i)
            if n == 1:
                eng.release([seqs.pop(0)])
                if compact:
                    eng.compact(seqs + [lone], 24)
            live = seqs + [lone]
            out.append(eng.decode_step(live, torch.tensor([s.tokens[-1] for s in live])))
    assert all(torch.equal(a, b) for a, b in zip(out[:3], out[3:]))
