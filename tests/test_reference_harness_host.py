"""What happens where the reference's own kernels were not built: the loader fails as any loader does, and the comparisons that
need it are skipped by a mark, unless the reference's sources are there and a build was to be expected."""
import types

import pytest

import conftest
from oracle import ref_cuda


def test_the_loader_raises_an_ordinary_error(monkeypatch, tmp_path):
    monkeypatch.setattr(ref_cuda, "_lib", None)
    monkeypatch.setattr(ref_cuda, "LIB_PATH", str(tmp_path / "libref_splat.so"))
    assert not ref_cuda.available()
    try:
        ref_cuda.lib()
    except OSError as e:
        assert "libref_splat.so" in str(e)
    except BaseException as e:      # a skip would end this test as skipped
        pytest.fail(f"{type(e).__name__} from a loader")
    else:
        pytest.fail("nothing to load, and no error")


class Item:
    def __init__(self, path, name):
        self.path, self.originalname, self.marks = types.SimpleNamespace(name=path), name, []

    def add_marker(self, mark):
        self.marks.append(mark)


@pytest.mark.parametrize("built, sources, skipped", [(True, True, False), (True, False, False), (False, True, False), (False, False, True)])
def test_comparisons_without_a_mark_of_their_own(monkeypatch, built, sources, skipped):
    monkeypatch.setattr(ref_cuda, "available", lambda: built)
    monkeypatch.setattr(ref_cuda, "reference_root", lambda: "somewhere" if sources else None)
    items = [Item("test_gpu_reference.py", name) for name in sorted(conftest.REFERENCE_COMPARISONS)]
    others = [Item("test_gpu_reference.py", "test_reference_known_answer_ranges_on_the_cuda_kernels"),
              Item("test_elsewhere.py", items[0].originalname)]
    conftest.pytest_collection_modifyitems(items + others)
    assert all(len(i.marks) == skipped for i in items) and not any(i.marks for i in others)
    assert all(m.name == "skip" and "not built" in m.kwargs["reason"] for i in items for m in i.marks)
