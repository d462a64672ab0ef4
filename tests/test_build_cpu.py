"""The link command of the torch binding."""
import os

from flashlite_b200 import build


def test_runtime_is_linked_from_where_it_is_loaded(monkeypatch, tmp_path):
    """The C++ runtime is named by its path: whether a linker's search path has the file is its compiler's affair."""
    commands = []
    monkeypatch.setattr(build, "_stale", lambda target, deps: True)
    monkeypatch.setattr(build, "_run", lambda cmd, log=None: commands.append(cmd) or "")
    monkeypatch.setattr(build, "BUILD", tmp_path)
    build.build_binding()
    link = next(c for c in commands if "-shared" in c)
    assert not [x for x in link if x.startswith("-l:")]
    runtime = [x for x in link if "libstdc++" in x]
    assert len(runtime) == 1 and os.path.isfile(runtime[0])


def test_runtime_of_the_process(tmp_path):
    maps = tmp_path / "maps"
    line = "7f0000000000-7f0000100000 r-xp 00000000 08:01 42   %s\n"
    maps.write_text(line % "/lib/libc.so.6" + line % "/odd place/libstdc++.so.6.0.33" + line % "/other/libstdc++.so.6")
    assert build.loaded_cxx_runtime(maps) == ["/odd place/libstdc++.so.6.0.33"]
    maps.write_text(line % "/lib/libc.so.6")
    assert build.loaded_cxx_runtime(maps) == []
    assert build.loaded_cxx_runtime(tmp_path / "none") == []
