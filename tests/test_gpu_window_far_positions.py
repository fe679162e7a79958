"""Window attention over a page table that reaches as far as positions do: 16 entries short of 2^31."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_paged import call, oracle, setup

pytestmark = pytest.mark.gpu

PAGE, WIDTH = 16, (2 ** 31 - 1) // 16


@pytest.fixture(scope="module")
def far_table():
    return torch.full((1, WIDTH), -1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("new,ratio", [(1, 4), (40, 1), (40, 8)])
@pytest.mark.parametrize("drafted", [False, True])
def test_the_last_positions(new, ratio, drafted, far_table):
    """The tokens in front of the table's end, with the keys that they would have at positions near 0."""
    near, last = 1000 + 40 - new, PAGE * WIDTH - 1
    far = last - new + 1
    assert (far - near) % (2 * PAGE) == 0
    x = setup([new], [near], 1, ratio, 64, PAGE, torch.bfloat16, False)
    if drafted:
        x["parents"] = (torch.arange(new, dtype=torch.int32, device="cuda") - 3).clamp(min=-1)
    want, want_lse, tol, lse_tol = oracle(x, [new], [near], 100, 0, 64 ** -0.5)
    pages = near // PAGE + -(-new // PAGE) + 1
    first = (far - near) // PAGE
    used = x["table"][0, :pages][: WIDTH - first]
    far_table.fill_(-1)
    far_table[0, first:first + used.numel()] = used
    y = dict(x, table=far_table, context=torch.tensor([far], dtype=torch.int32, device="cuda"))
    out, lse = call(y, 100, 0)
    assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= lse_tol).all()


@pytest.mark.parametrize("new,ratio", [(1, 4), (40, 1), (400, 8)])
@pytest.mark.parametrize("drafted", [False, True])
def test_lengths_behind_the_table(new, ratio, drafted, far_table):
    """Windows that lie behind it, from 2^31 on too: no keys."""
    x = setup([new], [0], 1, ratio, 64, PAGE, torch.bfloat16, False)
    if drafted:
        x["parents"] = torch.arange(new, dtype=torch.int32, device="cuda") - 1
    far_table.fill_(0)
    y = dict(x, table=far_table, context=torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    out, lse = call(y, 10, 0)
    assert not out.any() and (lse == float("-inf")).all()
