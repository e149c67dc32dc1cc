"""Requests that cannot go on beside requests that can: the others keep their tokens."""
from types import SimpleNamespace

import pytest
import torch

from serving.allocator import BlockAllocator
from serving.controls import RequestParams, sample_each
from serving.layers import SchedulerConfig
from serving.scheduler import Scheduler
from test_gpu_requests import VOCAB, Words, make_model, pool_of, prompts_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def plain():
    return make_model()


def scheduler(model, cfg, budget=None, blocks=64):
    alloc = BlockAllocator(blocks)
    sc = SchedulerConfig(max_num_seqs=8, max_num_batched_tokens=budget,
                         enable_chunked_prefill=True,
                         cudagraph_batch_sizes=[1, 2]) if budget else None
    return Scheduler(model, pool_of(cfg, blocks), alloc, SimpleNamespace(eos_token_id=-1),
                     block_size=16, temperature=1.0, top_k=1, top_p=1.0, sched_cfg=sc)


def run(sched, steps=200):
    """Steps until nothing is left: ({seq_id: tokens}, the errors that were raised)."""
    got, errors = {}, []
    while (sched.running or sched.waiting) and steps:
        steps -= 1
        try:
            for sid, tok, _ in sched.step():
                got.setdefault(sid, []).append(tok)
        except ValueError as e:
            errors.append(e)
    assert steps, "the scheduler does not get on"
    return got, errors


def alone(model, cfg, prompt, n, params=None):
    sched = scheduler(model, cfg)
    sched.add_request(prompt, n, params=params)
    return run(sched)[0][0]


class Ends(Words):
    """A grammar that allows nothing once its states are used up."""

    def mask(self):
        if len(self.took) == len(self.allowed):
            return torch.zeros(-(-VOCAB // 32), dtype=torch.int32)
        return super().mask()


@pytest.mark.parametrize("budget", [None, 16])
def test_a_dead_end_ends_its_request_alone(plain, budget):
    model, cfg = plain
    prompts = prompts_of([9, 20, 5, 31])
    greedy = RequestParams(temperature=0, repetition_penalty=1.2)
    want = {0: alone(model, cfg, prompts[0], 12), 1: alone(model, cfg, prompts[1], 12, greedy),
            3: alone(model, cfg, prompts[3], 12)}
    sched = scheduler(model, cfg, budget)
    dead = Ends([[3, 5, 7], [10, 11]])
    for p, r in zip(prompts, (None, greedy,
                              RequestParams(temperature=0, frequency_penalty=0.1, grammar=dead),
                              None)):
        sched.add_request(p, 12, params=r)
    got, errors = run(sched)
    assert len(got.pop(2)) == 2 and len(dead.took) == 2
    assert got == want
    assert len(errors) == 1 and "no token left" in str(errors[0])
    assert list(errors[0].failed) == [2]
    assert sched.alloc.num_free == sched.alloc.num_usable
    assert not sched._state and not sched._history._row


@pytest.mark.parametrize("budget", [None, 16])
@pytest.mark.parametrize("where", ["advance", "mask", "shape"])
def test_a_grammar_that_raises_ends_its_request_alone(plain, budget, where):
    model, cfg = plain
    prompts = prompts_of([9, 20, 5])
    want = [alone(model, cfg, prompts[0], 8), None, alone(model, cfg, prompts[2], 8)]

    class Breaks(Words):
        def mask(self):
            if len(self.took) == 2 and where == "mask":
                raise KeyError("no state")
            if len(self.took) == 2 and where == "shape":
                return torch.zeros(3, dtype=torch.int32)
            return super().mask()

        def advance(self, token):
            if len(self.took) == 2 and where == "advance":
                raise KeyError("no state")
            super().advance(token)

    sched = scheduler(model, cfg, budget)
    for p, r in zip(prompts, (None, RequestParams(temperature=0, grammar=Breaks([[3, 5], [4]])),
                              None)):
        sched.add_request(p, 8, params=r)
    got, errors = run(sched)
    assert [got[0], got[2]] == [want[0], want[2]]
    # the token that the grammar choked on was drawn and is handed out
    assert len(got[1]) == (3 if where == "advance" else 2)
    assert len(errors) == 1 and list(errors[0].failed) == [1]
    assert ("words" if where == "shape" else "no state") in str(errors[0])
    assert sched.alloc.num_free == sched.alloc.num_usable


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_penalties_past_the_types_range_stop_nobody(dtype):
    model, cfg = make_model(dtype)
    prompts = prompts_of([9, 20, 5, 12, 7])
    want = alone(model, cfg, prompts[0], 10)
    sched = scheduler(model, cfg)
    for p, r in zip(prompts, (None, RequestParams(repetition_penalty=1e-30),
                              RequestParams(temperature=0, frequency_penalty=-3e38),
                              RequestParams(presence_penalty=-1e5, top_p=0.9),
                              RequestParams(presence_penalty=3e38, frequency_penalty=3e38,
                                            grammar=Words([[5]])))):
        sched.add_request(p, 10, params=r)
    got, errors = run(sched)
    assert not errors and got[0] == want and all(len(got[i]) == 10 for i in range(5))
    assert got[4] == [5] * 10  # the only token it may take, whatever it costs


def test_a_vocabulary_past_the_draws_is_refused_when_a_request_is_added(plain):
    model = torch.nn.Module()
    model.lm_head = torch.nn.Linear(1, (1 << 20) + 1, device=DEV)
    sched = Scheduler(model, None, None, None)
    with pytest.raises(ValueError, match="logits"):
        sched.add_request([1], 2, params=RequestParams())
    sched.add_request([1], 2)


def test_a_draw_without_temperatures_is_refused():
    with pytest.raises(ValueError, match="temperature"):
        sample_each(torch.zeros(2, 8, device=DEV), None)
