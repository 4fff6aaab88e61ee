"""The build recipe: which objects of an earlier build are kept."""
import os


def test_an_object_is_kept_only_while_all_it_was_made_of_is_older(tmp_path):
    from cuml_b200 import build

    source, header, late = (str(tmp_path / f) for f in ("a.cu", "a.hpp", "late.hpp"))
    obj = str(tmp_path / "a.o")
    assert not build._object_current(obj, "recipe")
    for path in (source, header, late, obj):
        open(path, "w").close()
        os.utime(path, (100, 100))
    assert not build._object_current(obj, "recipe")  # nothing is known of it
    with open(obj + ".d", "w") as fh:
        fh.write(f"{obj} : {source} \\\n    {header}\n")
    with open(obj + ".recipe", "w") as fh:
        fh.write("recipe")
    assert build._object_current(obj, "recipe")
    assert not build._object_current(obj, "the same of another compiler")
    os.utime(late, (200, 200))
    assert build._object_current(obj, "recipe")  # it was not made of this
    os.utime(header, (200, 200))
    assert not build._object_current(obj, "recipe")
    os.utime(obj, (300, 300))
    assert build._object_current(obj, "recipe")
    os.remove(header)
    assert not build._object_current(obj, "recipe")


def test_the_library_is_older_than_a_header_that_no_list_names(tmp_path, monkeypatch):
    from cuml_b200 import build

    lib, src = tmp_path / "libb2fil.so", tmp_path / "csrc"
    src.mkdir()
    (src / "new.cuh").touch()
    (src / os.path.basename(build.TORCH_SOURCE)).touch()
    lib.touch()
    monkeypatch.setattr(build, "SRC", str(src))
    monkeypatch.setattr(build, "LIB", str(lib))
    monkeypatch.setattr(build, "TORCH_SOURCE", str(src / os.path.basename(build.TORCH_SOURCE)))
    far = os.path.getmtime(build.__file__) + os.path.getmtime(lib) + 1000
    os.utime(lib, (far, far))
    os.utime(build.TORCH_SOURCE, (far + 10, far + 10))
    assert build._lib_up_to_date()  # (the torch call path is not part of it)
    os.utime(src / "new.cuh", (far + 10, far + 10))
    assert not build._lib_up_to_date()
