"""Calls at the edges of the operators of a policy step on the GPU: plans that do not fit, rows of finished sequences, long prefixes, captured steps, losses under autograd's other modes."""
import math

import pytest
import torch

from tests.policy_step_oracle import attention, batch
from tests.test_policy_step_gpu import E, close  # noqa: F401   (the fixture)

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
