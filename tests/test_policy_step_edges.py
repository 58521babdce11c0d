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
