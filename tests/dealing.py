"""A fixture that makes every call deal its work in a given way, whatever the rule says (None: the rule's)."""
import pytest

DEALS = [None, (0, 1), (0, 3), (0, 8), (7, 1), (296, 1)]


@pytest.fixture
def deal(request, monkeypatch):
    from block_sparse_attention import cached_attn, window_attn

    def clear():
        cached_attn._cached_plan.cache_clear()
        window_attn._window_plan.cache_clear()
    if request.param is not None:
        monkeypatch.setattr(window_attn, "_deal_work", lambda *sizes: request.param)
    clear()
    yield request.param
    clear()
