"""A launch that blocks because the device's queue is full leaves other Python threads running."""
import threading
import time

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.rotary import rotary_table

pytestmark = pytest.mark.gpu


def calls(device):
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.zeros(1, 2, 64, device=device).half()
    cache = torch.zeros(2, 16, 2, 64, device=device).half()
    table, out = rotary_table(4, 64, device=device), torch.empty_like(q)
    slots = torch.zeros(1, dtype=torch.long, device=device)
    plan = (ints(0), ints(0, 1), ints(0)[None], ints(1), ints(1), ints(1), 1, 16)
    attend = (q, cache, cache, ints(0)[None], ints(0), ints(0, 1))
    return dict(rotary=lambda: fa.rotary(q, None, table, out_q=out),
                rotary_append=lambda: fa.rotary_append(q, q, q, table, None, slots, cache, cache, out_q=out),
                plan_cache_step=lambda: fa.plan_cache_step(*plan), tree_attention=lambda: fa.tree_attention(*attend, out=out))


@pytest.mark.parametrize("name", ["rotary", "rotary_append", "plan_cache_step", "tree_attention"])
def test_other_threads_run(cuda, name):
    call = calls(cuda)[name]
    call()
    torch.cuda.synchronize()
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.001)

    side = threading.Thread(target=tick)
    side.start()
    try:
        torch.cuda._sleep(3_000_000_000)  # 1.5 s and more of a kernel that only counts cycles
        begin = longest = time.perf_counter()
        longest = 0.0
        for _ in range(3000):
            before = time.perf_counter()
            call()
            longest = max(longest, time.perf_counter() - before)
            if time.perf_counter() - begin > 1.2:
                break
        end = time.perf_counter()
    finally:
        stop.set()
        side.join()
        torch.cuda.synchronize()
    if longest < 0.5:
        pytest.skip("the queue did not fill")
    inside = [begin, *(t for t in ticks if begin < t < end), end]
    gap = max(b - a for a, b in zip(inside, inside[1:]))
    assert gap < longest / 2
