"""build() compiles the reference's extension only where its sources are."""
import __graft_entry__ as entry


def test_an_empty_directory_is_no_reference(tmp_path):
    assert not entry.has_reference(str(tmp_path)) and not entry.has_reference(str(tmp_path / "nothing"))
    (tmp_path / "src" / "coresets" / "cuda" / "kernels").mkdir(parents=True)
    assert entry.has_reference(str(tmp_path))
