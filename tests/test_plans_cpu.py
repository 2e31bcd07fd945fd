"""CPU: which of the plans that calls keep for their shapes are given up."""
from splitd_flash_attn import rotary
from splitd_flash_attn.rotary import _Plans


def test_the_plan_unused_for_the_longest_time_goes(monkeypatch):
    monkeypatch.setattr(rotary, "_PLANS_MOST", 4)
    plans = _Plans()
    assert plans.find("decode") is None
    assert plans.keep("decode", "D") == "D"
    for n in range(100):  # prompts of ever new lengths between the decode steps
        assert plans.find(n) is None
        plans.keep(n, str(n))
        assert plans.find("decode") == "D" and len(plans) <= 4
    assert sorted(map(str, plans)) == ["97", "98", "99", "decode"]
    assert plans.find(96) is None and plans.find(98) == "98"


def test_plans_of_several_threads(monkeypatch):
    """Whatever comes in between, a plan that is found is the one for its key, and their number stays bounded."""
    import threading

    monkeypatch.setattr(rotary, "_PLANS_MOST", 8)
    plans, wrong = _Plans(), []

    def work(seed):
        for i in range(4000):
            key = (i * seed) % 13
            plan = plans.find(key)
            if plan is None:
                plan = plans.keep(key, ("plan", key))
            if plan != ("plan", key):
                wrong.append((key, plan))

    threads = [threading.Thread(target=work, args=(s,)) for s in (3, 5, 7, 11)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(plans) <= 8 + 4
