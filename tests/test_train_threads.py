"""Steps of one AdamW plan from several threads, the launch replaced by one that takes its time, on CPU."""
import threading
import time

import pytest


def test_each_step_has_its_own_rate_and_count(monkeypatch):
    import torch
    from omoknuni_small_b200 import capi
    capi.lib()
    plan = object.__new__(capi.AdamW)
    plan.device, plan.table, plan.cfg, plan.steps = torch.device("cpu"), (capi.TrainTensor * 1)(), capi.AdamWConfig(), 0
    plan._lock = threading.Lock()
    plan._ran_on = lambda stream: None
    seen = []

    def launch(device, fn, table, n, c):
        mine = (c.step, c.lr, c.grad_scale)
        for _ in range(5):
            time.sleep(0.001)                    # the interpreter goes to the other threads
            assert (c.step, c.lr, c.grad_scale) == mine
        seen.append(mine)
    monkeypatch.setattr(capi, "_launch_on", launch)
    scales = [torch.ones(1) for _ in range(6)]
    threads = [threading.Thread(target=lambda k=k: [plan.step(0.5 + k, grad_scale=scales[k]) for _ in range(5)]) for k in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert plan.steps == 30 and [s for s, _, _ in seen] == list(range(1, 31))
    assert all(p == scales[int(lr)].data_ptr() for _, lr, p in seen)
    with pytest.raises(capi.Error):
        plan.step(0.1, grad_scale=torch.ones(2))
    plan.step(0.1)                               # a refused step holds nothing up
    assert plan.steps == 31
