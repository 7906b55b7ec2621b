"""Which tests run where."""
import pytest

import conftest


class Item:
    def __init__(self, name):
        self.originalname, self.marks = name, []

    def add_marker(self, mark):
        self.marks.append(mark)


@pytest.mark.parametrize("device", [False, True])
def test_made_up_addresses_stay_off_a_device(monkeypatch, device):
    monkeypatch.setattr(conftest, "device_present", lambda: device)
    items = [Item(name) for name in sorted(conftest.MADE_UP_ADDRESSES)] + [Item("test_append_matches_reference")]
    conftest.pytest_collection_modifyitems(None, items)
    assert all([m.name for m in i.marks] == ["skip"] * device for i in items[:-1]) and items[-1].marks == []


@pytest.mark.parametrize("name", sorted(conftest.MADE_UP_ADDRESSES))
def test_names_are_those_of_tests(name):
    import test_kv_append
    import test_logits
    import test_prefix_attention
    assert sum(hasattr(m, name) for m in (test_kv_append, test_logits, test_prefix_attention)) == 1
