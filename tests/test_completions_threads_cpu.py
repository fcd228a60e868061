"""Completions of one prompt while other threads hand in requests."""
import sys
import threading

import pytest
import torch


def _engine(**kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    return InferenceEngine("gpt-tiny", device="cpu", **{"kv_block_size": 4, "num_kv_blocks": 64, "max_batch_size": 6, "max_batch_tokens": 512, **kw})


@pytest.fixture
def _threads_take_turns_often():
    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    yield
    sys.setswitchinterval(before)


def test_requests_that_come_while_a_prompt_is_looked_for(_threads_take_turns_often):
    eng = _engine()
    for _ in range(3000):                      # many that wait: looking through all of them takes long
        eng.add_request([9, 8, 7], 1, 0.0)
    stop, added = threading.Event(), []

    def more():
        while not stop.is_set() and len(added) < 30000:
            added.append(eng.add_request([5, 6], 1, 0.0))

    group = eng.add_requests([4, 5, 6, 7, 8], 4, 3, 0.0)
    eng.sched.step()
    first = group[0]
    eng.kv.allocate(first.req_id, 5), eng._prefill(first)
    for s in group[1:]:
        eng.kv.allocate(s.req_id, 5)
    threads = [threading.Thread(target=more) for _ in range(2)]
    for t in threads:
        t.start()
    try:
        for _ in range(300):
            for s in group[1:]:
                assert torch.equal(eng._prefill(s), first.prompt_logits)
    finally:
        stop.set()
        for t in threads:
            t.join()
    assert all(eng.kv.block_table(s.req_id)[:1] == eng.kv.block_table(first.req_id)[:1] for s in group[1:])


def test_a_completion_finds_its_prompt_whatever_stands_before_it():
    """Whoever had the prompt may end, be cancelled or lose its blocks: the others go on with what is there."""
    eng = _engine(max_batch_size=2)
    seqs = eng.add_requests([4, 5, 6, 7, 8, 9, 10, 11, 12], 6, 4, 0.0)
    spent = []
    while eng.has_work():
        before = eng.stats["prefill_tokens"]
        eng.step()
        spent.append(eng.stats["prefill_tokens"] - before)
    assert len({tuple(s.generated) for s in seqs}) == 1 and all(len(s.generated) == 4 for s in seqs)
    assert eng.kv.free_blocks == 64 and all(s.prompt_logits is None and s.prefix is None for s in seqs)
    assert sum(spent) <= 3 * 9                 # two at a time: once for each pair


def test_a_server_that_many_ask_at_once(_threads_take_turns_often):
    """Nobody's request ends in an error because others hand in theirs."""
    from llmctl_b200.serve.server import EngineLoop
    eng = _engine()
    loop, seqs = EngineLoop(eng), [[] for _ in range(3)]

    def ask(i):
        for k in range(40):
            seqs[i] += eng.add_requests([4 + i, 5, 6, 7, 8, 9], 3, 3, 0.0) if i else [eng.add_request([9, 8, 7 + k % 3], 3, 0.0)]
            loop.wake.set()

    loop.start()
    threads = [threading.Thread(target=ask, args=(i,)) for i in range(3)]
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for s in sum(seqs, []):
            assert s.done_event.wait(60)
    finally:
        loop.stop()
    assert loop.error is None and all(s.finish_reason in ("length", "stop") for s in sum(seqs, []))
    assert eng.kv.free_blocks == 64


def test_a_request_may_be_planned_as_soon_as_it_is_handed_in():
    """The engine's thread steps between the scheduler's taking a request and the return of the call that brings it."""
    eng = _engine()
    take = eng.sched.add_request
    eng.sched.add_request = lambda *a: (take(*a), eng.step())[0]
    seq = eng.add_request([9, 8, 7], 3, 0.0)
    assert len(seq.generated) == 1
    while eng.has_work():
        eng.step()
    assert len(seq.generated) == 3 and not eng.seqs
    refused = eng.add_request([1] * 400, 200, 0.0)          # more than the engine's tokens
    assert refused.finish_reason == "error" and not eng.seqs
