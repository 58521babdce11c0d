"""Operators of a policy step at their edges, on the CPU: room and order of plans, forks that do not fit."""
import random

import pytest
import torch

from twinkle_b200 import ops


def test_room_of_plans_of_groups():
    """Every plan whose sharing groups have two sequences or more fits; places that it does not use come first."""
    rng = random.Random(2)
    for _ in range(300):
        G, hkv, bs = rng.choice([1, 3, 4, 7, 16, 32, 42, 43, 64, 65, 128]), rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 64])
        sizes = [rng.choice([1, 2, 2, 3, 3, 5, 8, rng.randint(1, 130)]) for _ in range(rng.randint(1, 12))]
        blocks = [0 if n == 1 else rng.choice([0, 1, 3, rng.randint(0, 2000)]) for n in sizes]
        items, _ = ops._prefix_items(sizes, blocks, bs, G, hkv, 148)
        room = ops.prefix_items(sum(sizes), hkv, 'cpu', G)
        assert len(items) <= room <= ops.prefix_items(sum(sizes), hkv, 'cpu')
        plan = ops.shared_prefix(sizes, blocks, bs, G * hkv, hkv, device='cpu', items=room)
        places = plan.plan[:8 * room].view(room, 8)
        assert plan.items == room and (places[:room - len(items), 3] == 0).all() and places[room - len(items):].tolist() == items


def test_sharing_is_a_part_of_the_serving_subset():
    from twinkle_b200.ops import build
    names = lambda *parts: {p.rsplit('/', 1)[-1] for p in build._sources(parts)}  # noqa: E731
    assert names('sharing') - names() == {'cache_copy.cu', 'paged_shared.cu'} and 'losses.cu' not in names(*build._PARTS)
    with open(build._CSRC + '/bindings.cpp') as f:
        text = f.read()
    bound = text[text.index('TK_WITH_SHARING'):text.index('TK_WITH_CONVOLUTION')]
    assert all(f'm.def("{n}"' in bound for n in ('paged_attn_shared', 'paged_shared_split', 'cache_copy'))


def _engine_and(stack, n, **args):
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.sampler.engine import NativeEngine, _Seq
    cfg = preset(stack)
    eng = NativeEngine(build_model(cfg, device='cpu', dtype=torch.float32, seed=0), cfg, share_prompts=True, **{**dict(num_blocks=64, block_size=4, max_batch=8), **args})
    return eng, [_Seq(0, [3, 4, 5, 6, 7, 8], SamplingParams(max_tokens=4)) for _ in range(n)]


@pytest.mark.parametrize('what', ['has not run', 'other prompt', 'longer prompt', 'other adapter', 'has run', 'has tokens', 'twice'])
def test_forks_that_are_refused(what):
    eng, (a, b, c) = _engine_and('tiny-dense', 3)
    if what != 'has not run':
        eng.prefill([a])
    if what == 'other prompt':
        b.prompt = [9] * 6
    elif what == 'longer prompt':
        b.prompt = a.prompt + [1]
    elif what == 'other adapter':
        b.slot = 1
    elif what == 'has run':
        eng.prefill([b])
    elif what == 'has tokens':
        b.tokens.append(1)
    free, held = list(eng.cache.free), list(b.blocks)
    with pytest.raises(ValueError):
        eng.fork(a, [c, b, c] if what == 'twice' else [c, b])
    assert eng.cache.free == free and not eng.cache.sharers and b.blocks == held and c.blocks == [] and a.origin is None


@pytest.mark.parametrize('stack', ['tiny-dense', 'tiny-hybrid'])
def test_forks_of_a_sequence_that_has_gone_on(stack):
    """Keys and values of the prompt are still there; a state is not."""
    eng, (a, b, c) = _engine_and(stack, 3)
    eng.prefill([a])
    a.tokens.append(11)
    eng.grow([a])
    eng.decode_step([a], torch.tensor([11]))
    if stack == 'tiny-hybrid':
        with pytest.raises(ValueError, match='state'):
            eng.fork(a, [b])
        return
    eng.fork(a, [b])
    eng.prefill([c])
    for s in (b, c):
        s.tokens.append(12)
        eng.grow([s])
    x, y = (eng.decode_step([s], torch.tensor([12])) for s in (b, c))
    assert torch.allclose(x, y, atol=1e-5)


def test_routing_of_forks_is_that_of_the_prompt():
    eng, (a, b) = _engine_and('tiny-dense', 2)
    eng.prefill([a])
    a.routed = [torch.arange(9).view(9, 1)]
    a.tokens += [1, 2, 3]
    eng.fork(a, [b])
    assert b.routed[0].tolist() == [[i] for i in range(6)]


# heads, groups, shared tokens, own tokens, and what a layer of a captured step took on a B200: us together, us apart
MEASURED = [((32, 4, 128), [8], [1024], [256] * 8, 11.2, 9.1), ((32, 4, 128), [16], [1024], [256] * 16, 12.5, 17.4), ((32, 8, 64), [8] * 8, [64] * 8, [256] * 64, 17.3, 11.3),
            ((32, 8, 64), [64], [1024], [256] * 64, 19.9, 24.6), ((32, 8, 128), [64], [512], [256] * 64, 23.3, 35.0), ((12, 2, 128), [4], [512], [256] * 4, 9.7, 6.4),
            ((32, 8, 128), [4], [512], [256] * 4, 9.6, 7.6), ((32, 8, 128), [8], [512], [256] * 8, 10.4, 15.1), ((16, 8, 128), [2], [512], [256] * 2, 9.4, 18.7), ((8, 8, 128), [4], [1024], [256] * 4, 10.7, 33.3),
            ((16, 8, 128), [4], [496], [256] * 4, 9.6, 21.9), ((32, 8, 128), [2] + [1] * 62, [4096] + [0] * 62, [256] * 2 + [4352] * 62, 195.0, 167.2), ((32, 8, 64), [2] * 32, [512] * 32, [256] * 64, 30.2, 18.2),
            ((32, 8, 128), [2] * 32, [128] * 32, [256] * 64, 30.3, 24.5), ((32, 8, 128), [256], [1024], [256] * 256, 68.1, 119.1), ((12, 2, 128), [64], [128], [256] * 64, 11.6, 16.5)]


@pytest.mark.parametrize('heads,sizes,tokens,own,together,apart', MEASURED)
def test_the_faster_way_is_expected_to_be(heads, sizes, tokens, own, together, apart):
    a, b = ops.shared_times(sizes, [t // 16 for t in tokens], own, 16, *heads, device='cpu')
    assert (a < b) == (together < apart)


@pytest.mark.parametrize('heads,sizes,tokens,own,together,apart', MEASURED)
def test_an_engine_shares_where_it_pays(heads, sizes, tokens, own, together, apart):
    """By the groups and the lengths of its sequences; 0 for wherever pages are shared; never for a cache that the kernel does not take."""
    from twinkle_b200.data_format import SamplingParams
    from twinkle_b200.models import build_model, preset
    from twinkle_b200.sampler.engine import NativeEngine, _Seq
    cfg = preset('qwen3-8b', num_hidden_layers=1, hidden_size=64, intermediate_size=64, num_attention_heads=heads[0], num_key_value_heads=heads[1], head_dim=heads[2], vocab_size=64)
    eng = NativeEngine(build_model(cfg, device='cpu', dtype=torch.bfloat16, seed=0), cfg, num_blocks=4, share_prompts=True)
    seqs, at = [], 0
    for n, t in zip(sizes, tokens):
        group = [_Seq(0, [1] * (t or own[at + i] - 1), SamplingParams(), tokens=[1] * (own[at + i] if t else 1)) for i in range(n)]
        for s in group:
            s.origin, s.blocks = group[0] if n > 1 else None, [1] * ((s.length + 271) // 16)
        seqs += group
        at += n
    assert (eng._shared(seqs, len(seqs), captured=True) is not None) == (together < apart)
    if abs(apart - together - 9) > 6:
        assert (eng._shared(seqs, len(seqs)) is not None) == (together + 9 < apart)      # an eager step has to save the host's time too
    eng.share_from = 0
    assert eng._shared(seqs, len(seqs)) is not None
    eng.share_from, eng.dtype = 1.0, torch.float32
    assert eng._shared(seqs, len(seqs)) is None


def test_own_pages_are_cut_by_the_longest_own_part():
    """Not by what the widest row of the table leaves beside the shortest prefix: a sequence that shares nothing is its own part from its first token."""
    eng, seqs = _engine_and('tiny-dense', 5, num_blocks=2000, block_size=8)
    eng.share_from = 0
    for s, prompt, room in zip(seqs, (800, 800, 800, 400, 40), (10, 10, 12, 60, 6)):
        s.prompt, s.blocks = [1] * prompt, [1] * (prompt // 8 + room)
    for s in seqs[:3]:
        s.origin = seqs[0]
    assert eng._shared(seqs, 5).own == 8 * (50 + 60) and eng._shared(seqs[:3], 3).own == 8 * 12


def test_a_plan_is_made_again_when_answers_have_other_room():
    eng, seqs = _engine_and('tiny-dense', 3, num_blocks=2000, block_size=8)
    eng.share_from = 0
    for room in (12, 80):
        for s in seqs:
            s.prompt, s.blocks, s.origin = [1] * 800, [1] * (100 + room), seqs[0]
        assert eng._shared(seqs, 3).own == 8 * room
