"""What keeps the interpreter's full collections out of runs of steps: in the trainer, and the same in the benchmark."""
import ast
import gc
import os
from types import SimpleNamespace

import pytest

from legommenders_amd import trainer


def _trainer(step):
    policy = SimpleNamespace(epoch=1, epoch_batch=None, check_interval=0)
    t = object.__new__(trainer.Trainer)
    t.exp = SimpleNamespace(policy=policy, store=SimpleNamespace(patience=1, metric="GAUC"))
    t.steps_per_epoch, t.ts = 1, SimpleNamespace(step=step)
    return t


def test_training_leaves_what_was_there_out_of_collections():
    before, during = gc.get_freeze_count(), []

    def step():
        during.append((gc.get_freeze_count(), gc.isenabled()))
        raise KeyboardInterrupt
    with pytest.raises(KeyboardInterrupt):
        _trainer(step).train()
    assert during[0][0] > before + 10000 and during[0][1]
    assert gc.get_freeze_count() == 0                                                        # and gives it back, however it ends


def test_a_heap_that_the_caller_froze_stays_frozen():
    gc.freeze()
    try:
        n = gc.get_freeze_count()
        with trainer.frozen_heap():
            pass
        assert gc.get_freeze_count() >= n - 1000                                             # (objects that went by reference count are no longer in it)
    finally:
        gc.unfreeze()


def test_the_benchmark_times_the_same():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {n.id for n in ast.walk(ast.parse(open(os.path.join(root, "bench.py")).read())) if isinstance(n, ast.Name)}
    assert "frozen_heap" in names and "gc" not in names
