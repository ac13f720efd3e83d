"""What a step tells the prompt kernel of an 8-bit cache: the rows of its prompts, and the keys they hold."""

import numpy as np
import torch

from acorninfer_b200.cache.manager import CacheManager
from acorninfer_b200.engine.batch import StepEntry, pad_prefill_plan, plan_step
from acorninfer_b200.kernels import attention as attn
from acorninfer_b200.parts.base import KVNeeds


class Inputs:
    def __init__(self, plan):
        self.plan, self.extra = plan, {}


def planned(lens, window=None, P=16):
    """A step of rows (tokens held, tokens brought) over a group that keeps all keys and one of a window."""
    needs = {0: KVNeeds(2, 64), 1: KVNeeds(2, 64, window or 40)}
    manager = CacheManager(needs, {}, 400, P, 8, allocate=False)
    entries = []
    for i, (held, n) in enumerate(lens):
        rc = manager.open(i)
        for at in list(range(8, held, 8)) + [held]:
            manager.extend(rc, at)
            manager.commit(rc, at)
        manager.extend(rc, held + n)
        entries.append(StepEntry(rc, [1] * n, []))
    return manager, plan_step(entries, manager, attn.f8_step_arrays(8, 2))


def keys(plan, group, capturing, monkeypatch, P=16):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    return attn._f8_prompt_keys(Inputs(plan), group, plan.groups[group].block_table.shape[1] * P)


def test_rows_and_keys_of_a_mixed_step(monkeypatch):
    manager, plan = planned([(700, 1), (0, 300), (333, 33), (50, 31), (64, 32), (90, 2)])
    assert plan.extra["attention.f8_large_rows"].tolist() == [1, 2, 4]
    assert sorted(set(plan.extra["attention.f8_large"][:, 0].tolist())) == [1, 2, 4]
    assert keys(plan, 0, False, monkeypatch) == [300, 366, 96]
    # a window of 40: of 333 tokens held the first 18 pages are given back, of 64 the first one
    assert plan.groups[1].page_base.tolist()[2] == (333 - 40 + 1) // 16 and plan.groups[1].page_base.tolist()[4] == 1
    assert keys(plan, 1, False, monkeypatch) == [300, 366 - 18 * 16, 96 - 16]
    # what the table names covers them
    for gi, g in enumerate(plan.groups):
        assert all(k <= g.block_table.shape[1] * 16 for k in keys(plan, gi, False, monkeypatch))


def test_a_captured_step_takes_what_the_table_has_room_for(monkeypatch):
    manager, plan = planned([(50, 40)])
    padded = pad_prefill_plan(plan, manager.pad_pages, 16, attn.f8_step_arrays(8, 2))
    assert padded.extra["attention.f8_large_rows"].tolist() == [0] and padded.num_tokens == 64
    assert keys(padded, 0, True, monkeypatch) == [padded.groups[0].block_table.shape[1] * 16]
    assert keys(padded, 0, False, monkeypatch) == [50 + 64]


def test_steps_without_prompts(monkeypatch):
    _, plan = planned([(5, 1), (7, 31)])
    assert plan.extra["attention.f8_large_rows"].shape == (0,) and plan.extra["attention.f8_large_rows"].dtype == np.int32
    assert keys(plan, 0, False, monkeypatch) == []
