"""Calls with made-up addresses that pass every check reach no device: their tests are skipped where there is one."""
import pytest

from tests import conftest


class Item:
    def __init__(self, name, *marks):
        self.name, self.marks = name, [m.name for m in marks]

    def get_closest_marker(self, name):
        return name if name in self.marks else None

    def add_marker(self, mark):
        self.marks.append(mark.name)


@pytest.mark.parametrize("devices", [0, 1, 8])
def test_skipped_where_there_is_a_device(monkeypatch, devices):
    monkeypatch.setattr(conftest, "devices", lambda: devices)
    items = [Item("test_columns_of_one_row_are_apart"), Item("test_x", pytest.mark.no_gpu), Item("test_y"), Item("test_z", pytest.mark.gpu)]
    conftest.pytest_collection_modifyitems(items)
    assert ["skip" in item.marks for item in items] == [devices > 0, devices > 0, False, False]


def test_without_a_device_they_run():
    if conftest.devices():
        pytest.skip("there is one")
    from tests.test_rotate_validation_cpu import test_columns_of_one_row_are_apart
    test_columns_of_one_row_are_apart()
