"""Calls at the edges of the operators of a policy step on the GPU: plans that do not fit, rows of finished sequences, long prefixes, captured steps, losses under autograd's other modes."""
import math

import pytest
import torch

from tests.policy_step_oracle import attention, batch
from tests.test_policy_step_gpu import E, _policy_inputs, close  # noqa: F401   (the fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------- plans
BAD_ITEMS = {'more sequences than a tile has rows': {1: 33}, 'sequences behind the last': {0: 30}, 'a first sequence far away': {0: 2**31 - 1}, 'no sequences': {1: 0}, 'a first block far away': {2: 2**24},
             'a block that wraps': {2: 2**31 - 1}, 'blocks behind the prefix': {3: 9}, 'a slot behind the last': {5: 99}, 'a prefix wider than the table': {4: 2**20}, 'no tokens': {4: -5},
             'pages of a row before the first': {6: -1}, 'pages of a row behind the piece': {6: 40}}


@pytest.mark.parametrize('what', list(BAD_ITEMS))
def test_pieces_that_no_plan_has_are_left_out(E, what):  # noqa: F811
    """The error word says so; sequences of other groups have their results."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([33, 2], [320, 200], 20, 16, 16, 4, 128, device='cuda')      # up to 32 sequences a tile: 17 + 16
    plan = ops.shared_prefix(sizes, shared, 16, 16, 4)
    want, top = attention(*x)
    for at, value in BAD_ITEMS[what].items():
        plan.plan[at] = value
    out = ops.paged_attention_shared(*x, plan)
    torch.cuda.synchronize()
    assert E.read_and_clear_error() != 0
    close(out[33:], want[33:], top[33:])


@pytest.mark.parametrize('line', [(0, 2**31 - 1, 1, 0), (320, 2**31 - 1, 2**31 - 1, 0), (320, 0, 2**31 - 1, 0), (320, 0, 1, 2**31 - 1), (320, 0, 1, 125), (-1, 0, 1, 0), (320, -1, 1, 0), (320, 0, 1, -1)])
def test_lines_that_no_plan_has_are_not_followed(E, line):  # noqa: F811
    """Such a sequence reads all of its own pages."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([3, 2], [320, 200], 20, 16, 16, 4, 128, device='cuda')
    plan = ops.shared_prefix(sizes, shared, 16, 16, 4)
    plan.plan[plan.items * 8 + 4:plan.items * 8 + 8] = torch.tensor(line, dtype=torch.int32, device='cuda')
    close(ops.paged_attention_shared(*x, plan), *attention(*x))


def test_finished_sequences_stay_in_their_group(E):  # noqa: F811
    """Rows that were cleared when their sequence ended, the first of a tile of query rows among them; the first of a group is finished but still names the pages."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([40, 5], [256, 130], 20, 16, 32, 8, 128, device='cuda')      # two tiles of 20 sequences
    plan = ops.shared_prefix(sizes, shared, 16, 32, 8)
    done = [3, 20, 39, 41]
    x[3][done] = 0
    x[4][done + [0]] = 0
    out = ops.paged_attention_shared(*x, plan)
    close(out, *attention(*x))
    assert not out[done + [0]].any()


# --------------------------------------------------------------------- losses
def test_kl_term_of_any_size(E):  # noqa: F811
    """One token alone, ratio one and no advantage.  Its loss is e^d − d − 1: up to |d| = 1 a series with a rounded sum and two products (3.5 roundings of 2^-24), beyond that e^d − 1 with an
    error of at most 2^-23 of itself, less d: 5.4 · 2^-24 at e^d − 1 = 2.  Its derivative 1 − e^d has the series' error times rest / (e^d − 1) < 0.6 and a rounding, or 2^-23."""
    from twinkle_b200 import ops
    d = torch.cat([torch.linspace(-2, 2, 401), *(c + torch.linspace(-0.02, 0.02, 41) for c in (-1, -0.5, 0.5, 1)), torch.tensor([-15.0, -4.0, 4.0, 15.0])]).cuda()
    zero, one = torch.zeros(1, device='cuda'), torch.ones(1, len(d), dtype=torch.bool, device='cuda')
    wide = d.double()
    rest = torch.expm1(wide) - wide
    rest = torch.where(wide.abs() < 0.1, sum(wide**k / math.factorial(k) for k in range(2, 12)), rest)
    got = torch.stack([ops.policy_loss(zero[None], one[:, :1], zero, None, x.view(1, 1), beta=1.0)[0] for x in d]).double()
    assert ((got - rest).abs() <= 2**-21.5 * rest).all()
    lp = torch.zeros(1, len(d), device='cuda', requires_grad=True)
    g = torch.autograd.grad(ops.policy_loss(lp, one, zero, None, d[None], beta=1.0, reduce='sum')[0], lp)[0][0].double()
    assert ((g + torch.expm1(wide)).abs() <= 2**-22 * torch.expm1(wide).abs()).all()


def test_kl_gradient_of_tokens_that_the_reference_rules_out(E):  # noqa: F811
    """d = −∞ and far below: e^d − 1 is −1."""
    from twinkle_b200 import ops
    lp = torch.full((1, 4), -1.0, device='cuda', requires_grad=True)
    ref = torch.tensor([[-math.inf, -1e9, -200.0, -1.0]], device='cuda')
    loss = ops.policy_loss(lp, torch.ones(1, 4, dtype=torch.bool, device='cuda'), torch.zeros(1, device='cuda'), None, ref, beta=0.5, reduce='sum')[0]
    assert torch.autograd.grad(loss, lp)[0].tolist() == [[0.5, 0.5, 0.5, 0.0]] and float(loss.detach()) == math.inf


def test_ratios_are_those_of_the_exponential(E):  # noqa: F811
    """An exponential is off by at most 2^-23 of itself; the token's other factors are one."""
    from twinkle_b200 import ops
    l = torch.linspace(-19, 19, 5000, device='cuda')[None]
    for ratio, x, old in (('token', l, torch.zeros_like(l)), ):
        lp = x.clone().requires_grad_()
        loss, _ = ops.policy_loss(lp, torch.ones_like(l, dtype=torch.bool), torch.ones(1, device='cuda'), old, ratio=ratio, epsilon=1.0, epsilon_high=1e9, reduce='sum')
        g = torch.autograd.grad(loss, lp)[0].double()
        assert ((g + x.double().exp()).abs() <= 2**-22.9 * x.double().exp()).all()


def test_soft_gate_far_from_one(E):  # noqa: F811
    """The gate times what it leaves of one: e^-|z| (1 + e^-|z|)^-2 with z = τ (r − 1), |z| up to 40.  r − 1 is within 3 · 2^-24 (1.5 · 2^-23 of itself), so z, a product, within 4 · 2^-24 |z|; e^-|z| is
    off by that and 2^-23, the two quotients, the sum (met twice) and the products by a rounding each, the ratio by 2^-23: 4 |z| + 12 roundings of 2^-24."""
    from twinkle_b200 import ops
    r = torch.cat([torch.linspace(0.01, 0.99, 200), torch.linspace(1.01, 41, 800)]).double()
    lp = r.log().float().cuda()[None].requires_grad_()
    old, one = torch.zeros_like(lp), torch.ones_like(lp, dtype=torch.bool)
    g = torch.autograd.grad(ops.policy_loss(lp, one, torch.ones(1, device='cuda'), old, surrogate='soft', reduce='sum')[0], lp)[0].double()
    x = lp.detach().double()
    z = torch.expm1(x)
    e = torch.exp(-z.abs())
    want = -4 * e / (1 + e)**2 * x.exp()
    assert ((g - want).abs() <= (4 * z.abs() + 12) * 2**-24 * want.abs()).all()


# -------------------------------------------------------------- loss classes
@pytest.mark.parametrize('where', ['object', 'class', 'base'])
def test_replaced_rules_are_followed(E, where, monkeypatch):  # noqa: F811
    from twinkle_b200 import loss as L
    x = _policy_inputs(4, 50, 15)
    obj = L.SAPOLoss() if where == 'base' else L.GRPOLoss()
    call = lambda: obj({'labels': x['labels']}, {'logps': x['logps']}, old_logps=x['logps'], advantages=[1.0] * 4)['loss']  # noqa: E731
    before = E.launch_count()
    call()
    assert E.launch_count() > before
    if where == 'object':
        monkeypatch.setattr(obj, '_surrogate', lambda ratio, adv, logps: -3.0 * ratio * adv)
    elif where == 'class':
        monkeypatch.setattr(L.GRPOLoss, '_surrogate', lambda self, ratio, adv, logps: -3.0 * ratio * adv)
    else:
        monkeypatch.setattr(L.GRPOLoss, '_aggregate', lambda self, per_token, mask, **k: 3.0 * (per_token * mask).sum() / mask.sum())
    before = E.launch_count()
    got = float(call())
    # a token costs −r A = −1 (SAPO: −σ(0) · 4 = −2) times three; a row without tokens nothing
    rows = float(((x['labels'] != -100).any(-1)).float().mean())
    assert E.launch_count() == before and got == pytest.approx(-6.0 if where == 'base' else -3.0 * rows, abs=1e-5)


@pytest.mark.parametrize('name', ['_seq_logps', '_align_ref', '_nll'])
def test_replaced_parts_of_a_preference_loss_are_followed(E, name, monkeypatch):  # noqa: F811
    from twinkle_b200 import loss as L
    x = _policy_inputs(4, 50, 15)
    inputs, outputs, extra = {'labels': x['labels']}, {'logps': x['logps']}, dict(ref_logps=x['ref'])
    obj = L.DPOLoss(sft_weight=0.5)
    clean = float(obj(inputs, outputs, **extra)['loss'])
    real = getattr(obj, name)
    twice = {'_seq_logps': lambda *a: (lambda r: (r[0], r[1], 2 * r[2]))(real(*a)), '_align_ref': lambda *a: 2 * real(*a), '_nll': lambda *a: 2 * real(*a)}[name]
    monkeypatch.setattr(obj, name, twice)
    changed = float(obj(inputs, outputs, **extra)['loss'])
    on_cpu = float(obj({'labels': x['labels'].cpu()}, {'logps': x['logps'].cpu()}, ref_logps=x['ref'].cpu())['loss'])
    assert abs(changed - clean) > 1e-3 and changed == pytest.approx(on_cpu, rel=1e-4)


def _class_loss(name, x, logps, labels, **kwargs):
    from twinkle_b200 import loss as L
    extra = dict(old_logps=x['old'], advantages=[1.0, -0.5, 0.3, 2.0]) if name == 'GRPOLoss' else dict(ref_logps=x['ref'])
    extra = {n: v.to(logps.device) if torch.is_tensor(v) else v for n, v in {**extra, **kwargs}.items()}
    return getattr(L, name)()({'labels': labels}, {'logps': logps}, **extra)['loss']


@pytest.mark.parametrize('name', ['GRPOLoss', 'DPOLoss', 'SimPOLoss'])
def test_labels_may_be_written_again_before_the_backward_pass(E, name):  # noqa: F811
    """A buffer that the next micro-batch fills, and one of inference mode."""
    x = _policy_inputs(4, 50, 15)
    lp = x['logps'].clone().requires_grad_()
    want, = torch.autograd.grad(_class_loss(name, x, lp, x['labels'].clone()), lp)
    labels = x['labels'].clone()
    loss = _class_loss(name, x, lp, labels)
    labels.fill_(-100)
    assert torch.equal(torch.autograd.grad(loss, lp)[0], want)
    with torch.inference_mode():
        labels = x['labels'].clone()
    assert torch.equal(torch.autograd.grad(_class_loss(name, x, lp, labels), lp)[0], want)


@pytest.mark.parametrize('name', ['GRPOLoss', 'DPOLoss', 'ORPOLoss'])
@pytest.mark.parametrize('dtype', [torch.bool, torch.int32, torch.float32])
def test_labels_of_other_types_mean_what_they_mean_on_the_cpu(E, name, dtype):  # noqa: F811
    """A truth value is no mask here: both differ from the index that is ignored."""
    x = _policy_inputs(4, 50, 15)
    x['labels'][2, 3] = 7
    labels = (x['labels'] != -100) if dtype == torch.bool else x['labels'].to(dtype)
    got = [float(_class_loss(name, x, x['logps'].to(d), labels.to(d))) for d in ('cuda', 'cpu')]
    assert got[0] == pytest.approx(got[1], rel=1e-5)


@pytest.mark.parametrize('shape', [(1, 50), (1, 30), (2, ), (4, 1), (4, 50)])
@pytest.mark.parametrize('kind', ['sigmoid', 'ipo'])
def test_references_for_several_rows_are_spread(E, shape, kind):  # noqa: F811
    """One row of reference log-probs for all, two sums for all pairs."""
    from twinkle_b200 import loss as L
    x = _policy_inputs(4, 50, 15)
    ref = torch.linspace(-2, -0.5, math.prod(shape)).view(shape)
    got = [float(L.DPOLoss(loss_type=kind)({'labels': x['labels'].to(d)}, {'logps': x['logps'].to(d)}, ref_logps=ref)['loss']) for d in ('cuda', 'cpu')]
    assert got[0] == pytest.approx(got[1], rel=1e-5)


CLASSES = ['GRPOLoss', 'GSPOLoss', 'SAPOLoss', 'DPOLoss', 'SimPOLoss', 'CPOLoss', 'ORPOLoss']


def _both(name, f):
    """``f(loss as a function of log-probs, log-probs)`` of a class on the GPU in fp32 and on the CPU in fp64."""
    from twinkle_b200 import loss as L
    x = _policy_inputs(4, 50, 15)
    x['labels'][2, 3] = 7
    got = []
    for device, dtype in (('cuda', torch.float32), ('cpu', torch.float64)):
        y = {n: t.to(device) if n == 'labels' else t.to(device, dtype) for n, t in x.items()}
        kw = dict(old_logps=y['old'], ref_logps=y['ref'], advantages=y['adv']) if issubclass(getattr(L, name), L.GRPOLoss) else dict(ref_logps=y['ref'])
        obj = getattr(L, name)(**(dict(beta=0.1) if 'old_logps' in kw else {}))
        got.append(f(lambda lp: obj({'labels': y['labels']}, {'logps': lp}, **kw)['loss'], y['logps'].clone()).double().cpu())
    # sums of 50 terms in fp32, each off by a few roundings of 2^-24
    assert torch.isfinite(got[0]).all() and (got[0] - got[1]).abs().max() <= 2**-17 * got[1].abs().max()
    return got[0]


@pytest.mark.parametrize('name', CLASSES)
def test_gradients_of_gradients(E, name):  # noqa: F811
    def second(f, lp):
        lp.requires_grad_()
        g, = torch.autograd.grad(3.0 * f(lp), lp, create_graph=True)
        return torch.autograd.grad((g * torch.linspace(0, 1, g.numel(), device=g.device, dtype=g.dtype).view(g.shape)).square().sum(), lp)[0]

    assert _both(name, second).abs().sum() > 0


@pytest.mark.parametrize('name', CLASSES)
def test_losses_in_functional_transforms(E, name):  # noqa: F811
    _both(name, lambda f, lp: torch.func.grad(f)(lp))
    _both(name, lambda f, lp: torch.func.jvp(f, (lp, ), (torch.ones_like(lp), ))[1])


@pytest.mark.parametrize('name', CLASSES)
def test_several_gradients_of_a_loss_at_once(E, name):  # noqa: F811
    def batched(f, lp):
        lp.requires_grad_()
        return torch.autograd.grad(f(lp), lp, torch.tensor([1.0, -2.0, 0.5], device=lp.device, dtype=lp.dtype), is_grads_batched=True)[0]

    _both(name, batched)


def test_gradients_by_entropies_and_of_changed_inputs(E):  # noqa: F811
    from twinkle_b200 import ops
    x = _policy_inputs(4, 50, 15)
    lp, en = x['logps'].clone().requires_grad_(), x['ent'].clone().requires_grad_()
    call = lambda **k: ops.policy_loss(lp, x['labels'], x['adv'], x['old'], entropies=en, entropy_coef=0.1, **k)[0]  # noqa: E731
    first = torch.autograd.grad(call(twice=True), (lp, en), create_graph=True)
    plain = torch.autograd.grad(call(), (lp, en))
    assert all((a - b).abs().max() <= 2**-20 * b.abs().max() for a, b in zip(first, plain)) and first[0].requires_grad
    only, = torch.autograd.grad(call(twice=True), en, create_graph=True)
    assert (only - plain[1]).abs().max() <= 2**-20 * plain[1].abs().max()
    loss = call(twice=True)
    x['old'].zero_()                       # what a first gradient does not need, a second would
    assert torch.equal(torch.autograd.grad(loss, lp, retain_graph=True)[0], plain[0])
    with pytest.raises(RuntimeError, match='inplace'):
        torch.autograd.grad(loss, lp, create_graph=True)
    with pytest.raises(RuntimeError, match='one gradient'):
        torch.autograd.grad(call(), lp, torch.ones(2, device='cuda'), is_grads_batched=True)


@pytest.mark.parametrize('dtype', [torch.int64, torch.int32, torch.bool, torch.float64])
def test_operands_of_other_types_are_converted(E, dtype):  # noqa: F811
    from twinkle_b200 import ops
    x = _policy_inputs(4, 50, 15)
    adv, near = torch.tensor([[1], [0], [1], [1]], device='cuda'), (x['logps'] < -1).to(dtype)
    args = dict(beta=0.1, entropy_coef=0.1)
    want = ops.policy_loss(x['logps'], x['labels'], adv[:, 0].float(), near.float(), near.float(), near.float(), **args)
    for a in (adv[:, 0], adv.expand(4, 50)):
        got = ops.policy_loss(x['logps'], x['labels'], a.to(dtype), near, near, near, **args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(ops.preference_loss(x['logps'], x['labels'], near)[0], ops.preference_loss(x['logps'], x['labels'], near.float())[0])


# ------------------------------------------------------------- captured steps
def _small(num_attention_heads=8, num_key_value_heads=2, **args):
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.sampler.engine import NativeEngine
    cfg = preset('qwen3-8b', num_hidden_layers=2, hidden_size=512, intermediate_size=1024, num_attention_heads=num_attention_heads, num_key_value_heads=num_key_value_heads, vocab_size=1024)
    eng = NativeEngine(build_model(cfg, device='cuda', dtype=torch.bfloat16, seed=0), cfg, share_prompts=True, **args)
    eng.share_from = 0
    return eng


def test_captured_steps_are_laid_out_as_eager_ones(E, monkeypatch):  # noqa: F811
    """How many warps join a head and how far own pages are cut follow the plan and the table, not what was captured first; a shrinking group takes few captures."""
    from twinkle_b200 import ops
    from twinkle_b200.data_format import SamplingParams
    real, seen = ops.paged_attention_shared, []

    def noted(q, k, v, table, lens, prefix, scale=None):
        room = prefix.own if getattr(prefix, 'own', -1) >= 0 else (table.shape[1] - prefix.shared) * prefix.block_size
        seen.append((prefix.pieces > 8, min(8, (room + 255) // 256)))
        return real(q, k, v, table, lens, prefix, scale)

    monkeypatch.setattr(ops, 'paged_attention_shared', noted)
    prompts = [[(7 * i + 3) % 900 for i in range(3000)], [(3 * i + 1) % 900 for i in range(2200)]]
    laid, answers = [], []
    for graphs in (True, False):
        eng = _small(num_blocks=1000, block_size=16)
        eng.use_cuda_graphs = graphs
        seen.clear()
        res = eng.generate(prompts, [SamplingParams(max_tokens=n, temperature=0.0, num_samples=3) for n in (9, 6)])
        laid.append(set(seen))
        answers.append([s.tokens for r in res for s in r.sequences])
        assert bool(eng._graphs) == graphs
    assert laid[0] == laid[1] and any(many for many, _ in laid[0]) and any(runs < 8 for _, runs in laid[0])
    assert [a[:1] for a in answers[0]] == [a[:1] for a in answers[1]]


def test_calls_with_other_plans_of_the_same_room(E):  # noqa: F811
    """A plan with places that it does not use gives what the plan without them gives, bit for bit."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([5, 2], [1500, 90], 30, 16, 16, 4, 128, seed=1, device='cuda')
    plan, room = (ops.shared_prefix(sizes, shared, 16, 16, 4, items=n) for n in (0, 90))
    assert room.items > plan.items
    out = ops.paged_attention_shared(*x, plan)
    assert torch.equal(out, ops.paged_attention_shared(*x, room))
    wide = torch.cat([x[3], torch.zeros(7, 300, dtype=torch.int32, device='cuda')], 1)
    own = (x[3].shape[1] - plan.shared) * 16
    assert torch.equal(out, ops.paged_attention_shared(*x[:3], wide, x[4], room._replace(own=own)))


def test_steps_stay_captured_where_shared_ones_cannot_be(E, monkeypatch):  # noqa: F811
    """A captured step over shared prompts that finds no memory costs the sharing, not the capture of plain steps."""
    from twinkle_b200 import ops
    from twinkle_b200.data_format import SamplingParams
    prompts, params = [[(7 * i + 3) % 900 for i in range(400)]], [SamplingParams(max_tokens=6, temperature=0.0, num_samples=3)]
    want = _small(num_blocks=200).generate(prompts, params)

    def full(*args):
        raise torch.cuda.OutOfMemoryError('no memory')

    monkeypatch.setattr(ops, 'paged_attention_shared', full)
    eng = _small(num_blocks=200)
    res = eng.generate(prompts, params)
    assert eng.use_cuda_graphs and eng._graphs and not any(k[2] for k in eng._graphs)
    assert [s.tokens[:1] for s in res[0].sequences] == [s.tokens[:1] for s in want[0].sequences] and sorted(eng.cache.free) == list(range(1, 200))


# --------------------------------------------------------------- long prefixes
@pytest.mark.parametrize('sizes,prompts,bs,hq,hkv,D', [([3], [32760], 16, 8, 1, 128), ([2], [40000], 64, 4, 1, 64), ([2, 1, 3], [9000, 30, 7000], 16, 16, 2, 128)])
def test_prefixes_of_many_pieces(E, sizes, prompts, bs, hq, hkv, D):  # noqa: F811
    """Over 32 pieces a warp, over 128 a head, joined by four warps (the plan's own choice) and by one."""
    from twinkle_b200 import ops
    x, sizes, shared = batch(sizes, prompts, 40, bs, hq, hkv, D, device='cuda')
    plan = ops.shared_prefix(sizes, shared, bs, hq, hkv)
    assert plan.pieces > (32 if hkv > 1 else 100)
    want = attention(*x)
    for p in (plan, plan._replace(pieces=0)):
        close(ops.paged_attention_shared(*x, p), *want)


def test_a_prefix_in_pieces_of_one_block(E):  # noqa: F811
    """160 pieces a head, more than any plan of this GPU has."""
    from twinkle_b200 import ops
    x, sizes, shared = batch([2], [160 * 128 + 5], 20, 16, 8, 1, 128, device='cuda')
    items, lines = [[0, 2, i, 1, shared[0] * 16, i, 0, 0] for i in range(160)], [[shared[0] * 16, 0, 160, 8 * b] for b in range(2)]
    numbers = torch.tensor([n for part in items + lines for n in part], dtype=torch.int32, device='cuda')
    plan = ops.shared_prefix(sizes, shared, 16, 8, 1)._replace(plan=numbers, items=160, slots=160, pieces=160)
    want = attention(*x)
    for p in (plan, plan._replace(pieces=0)):
        close(ops.paged_attention_shared(*x, p), *want)


def test_captured_steps_behind_a_long_prompt(E):  # noqa: F811
    """Captured and eager steps of a group behind 20k tokens, against sequences that read their pages for themselves."""
    from twinkle_b200.sampler.engine import _Seq
    from twinkle_b200.data_format import SamplingParams
    prompt, steps = [(7 * i + 3) % 900 for i in range(20000)], {}
    for how in ('captured', 'eager', 'apart'):
        eng = _small(8, 1, num_blocks=1400)
        eng.use_cuda_graphs, eng.share_prompts = how == 'captured', how != 'apart'
        seqs = [_Seq(0, prompt, SamplingParams(max_tokens=8)) for _ in range(5)]
        eng.prefill(seqs[:1])
        eng.fork(seqs[0], seqs[1:])
        steps[how] = []
        for n in range(3):
            for i, s in enumerate(seqs):
                s.tokens.append((37 * n + 11 * i) % 900)
            steps[how].append(eng.decode_step(seqs, torch.tensor([s.tokens[-1] for s in seqs], device='cuda')).clone())
        eng.release(seqs)
        assert bool(eng._graphs) == (how == 'captured')
    for a, b, c in zip(*(steps[n] for n in ('captured', 'eager', 'apart'))):
        assert (a - c).norm() / c.norm() < 2e-2 and (b - c).norm() / c.norm() < 2e-2


def test_sharing_on_a_subset_without_it_is_refused(E, monkeypatch):  # noqa: F811
    from types import SimpleNamespace
    from twinkle_b200 import ops
    monkeypatch.setattr(ops, 'ext', lambda: SimpleNamespace())
    with pytest.raises(RuntimeError, match='sharing'):
        _small(num_blocks=20)
