"""The node pools' default budget (selfplay.pool_budget)."""
from citadels_self_play_amd import selfplay


def test_pool_budget_is_the_same_from_search_to_search(monkeypatch):
    """Free memory as counted before searches of one process, their pools cached in between: one budget."""
    monkeypatch.setattr(selfplay, "_budgets", {})
    seen = [307_299_876_864, 307_780_124_672, 307_683_655_680, 307_692_065_280, 307_908_050_944, 307_299_876_864]
    first = int(selfplay.POOL_FRAC * seen[0])
    assert [selfplay.pool_budget(n) for n in seen] == [first] * len(seen)


def test_pool_budget_follows_the_memory(monkeypatch):
    """Another device, or memory that others took or gave back: a budget of its own."""
    monkeypatch.setattr(selfplay, "_budgets", {})
    share = lambda n: int(selfplay.POOL_FRAC * n)  # noqa: E731
    for dev, n in (("cuda:0", 300 << 30), ("cuda:1", 298 << 30), ("cuda:0", 200 << 30), ("cuda:0", 5 << 20), ("cuda:0", 300 << 30)):
        assert selfplay.pool_budget(n, dev) == share(n)
    assert selfplay.pool_budget(298 << 30, "cuda:0") == share(300 << 30)
    assert selfplay.pool_budget(299 << 30, "cuda:1") == share(298 << 30)
