"""plan_compact and the scheduler: sequences that a scheduler runs, or caches as a prefix, are refused with nothing
changed; forks of them and other sequences are not."""
import numpy as np

from atomflow_amd import AF_ERR_BAD_SEQUENCE, kv


def state(bm, seqs):
    return bm.num_free_blocks(), [bm.seq_table(s) for s in seqs]


def test_sequences_of_a_scheduler():
    bm = kv.BlockManager(64, 8)
    mine = bm.seq_create()
    bm.seq_extend(mine, 30)
    sched = kv.Scheduler(bm, 4, 64, 32, max_cached_prefixes=2)
    sched.add_request(1, 20, 6, prefix_key=5, prefix_len=12)
    sched.add_request(2, 9, 6)
    for _ in range(3):
        sched.step()
    theirs = [s for s in range(8) if s != mine and bm.seq_len(s) >= 0]
    assert len(theirs) == 3  # two requests and the cached prefix
    before = state(bm, theirs + [mine])
    for s in theirs:
        assert bm.plan_compact([s], [[1, 3]]) == AF_ERR_BAD_SEQUENCE
        assert bm.plan_compact([mine, s], [[2], [0]]) == AF_ERR_BAD_SEQUENCE
    assert state(bm, theirs + [mine]) == before
    # a request that is admitted onto the cached prefix
    sched.add_request(3, 15, 2, prefix_key=5, prefix_len=12)
    plan = sched.step()
    hit = [c[1] for c in plan["prefill"]]
    assert len(hit) == 1 and bm.plan_compact(hit, [[0]]) == AF_ERR_BAD_SEQUENCE
    # the scheduler's own go on, and a fork of one is the caller's
    fork = bm.seq_fork(theirs[0])
    length = bm.seq_len(fork)
    plan = bm.plan_compact([fork, mine], [np.arange(1, length), [2, 29]])
    assert isinstance(plan, dict) and bm.seq_len(fork) == length - 1 and bm.seq_len(mine) == 2
    assert bm.seq_len(theirs[0]) == length
    for _ in range(12):
        sched.step()
    assert bm.seq_len(theirs[0]) < 0 and bm.seq_len(fork) == length - 1  # the requests have ended
    bm.close()
