"""What the device reports of a call on the 8-bit cache (needs a B200): one bit for each kind, no bit hiding another.

The waits run out because they are given no polls, as in test_gpu_bounded_wait.py: no copy or product is in
flight that the kernel does not wait for, and the context stays usable."""
import pytest
import torch

from kv8_helpers import Pool

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_polls(pkg, monkeypatch):
    monkeypatch.setenv("BZB_KV8_ATTENTION", "many")
    yield pkg.set_debug_kv8_polls
    pkg.set_debug_kv8_polls(-1)


@pytest.mark.parametrize("hd,L,new", [(64, 200, 40), (128, 300, 150), (64, 5000, 1)])  # (the last one with ranges)
def test_a_wait_that_runs_out_is_reported_and_recovered(pkg, no_polls, hd, L, new):
    pool = Pool(pkg, [L], 2, hd, 64, seed=1, fill=[L])
    batch = pool.batch([new], [L])
    q = torch.randn((new, 8, hd), device="cuda").half()
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    pool.cache.attention(batch, q, want, 0.1)
    pool.cache.check()
    no_polls(0)
    pool.cache.attention(batch, q, got, 0.1)
    with pytest.raises(RuntimeError, match="wait inside the attention ran out"):
        pool.cache.check()
    pool.cache.check()  # reported once
    no_polls(-1)
    pool.cache.attention(batch, q, got, 0.1)
    pool.cache.check()
    assert torch.equal(got, want)


@pytest.mark.parametrize("order", ["page first", "wait first"])
def test_neither_report_hides_the_other(pkg, no_polls, order):
    lens = [40, 40]
    pool = Pool(pkg, lens, 2, 64, seed=2, fill=lens)
    q = torch.randn((60, 4, 64), device="cuda").half()
    good, bad = pool.batch([30, 30], lens), pool.batch([30, 30], lens)
    bad._held[2][1] = -1
    calls = [lambda: pool.cache.read(bad, *(torch.empty((60, 2, 64), device="cuda") for _ in range(2))),
             lambda: pool.cache.attention(good, q, torch.empty_like(q), 0.1)]
    no_polls(0)
    for call in calls if order == "page first" else calls[::-1]:
        call()
    assert int(pool.cache.status.item()) == 3
    with pytest.raises(RuntimeError, match="out of range.*ran out"):
        pool.cache.check()
    pool.cache.check()
