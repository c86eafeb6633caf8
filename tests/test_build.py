"""The build's rules for what is out of date, with the compilers replaced by a stub (no GPU, no compiler)."""

import os

import pytest

from fermix_b200 import build


class Tree:
    """A source tree of its own and a stub that writes what a command names behind -o; commands on a name in `failing` fail."""

    def __init__(self, path, monkeypatch):
        self.path, self.failing, self.ran = path, set(), []
        for d in ("csrc", "include", "lib"):
            (path / d).mkdir()
        self.files = [path / "csrc" / n for n in ("one.cu", "two.cu", "all.cuh", "torch_binding.cpp")] + [path / "include" / "args.h"]
        for f in self.files:
            f.write_text("")
        self.clock = 1_000_000_000
        out, obj = path / "lib", path / "lib" / "obj"
        for name, value in dict(CSRC=path / "csrc", INCLUDE=path / "include", OUT_DIR=out, OBJ_DIR=obj, OUT=out / "library.so",
                                BINDING=path / "csrc" / "torch_binding.cpp", BINDING_OBJ=obj / "torch_binding.o",
                                BINDING_OUT=out / "binding.so", BINDING_FOR=out / "binding.for", __file__=path / "csrc" / "all.cuh").items():
            monkeypatch.setattr(build, name, str(value), raising=False)
        monkeypatch.setattr(build, "_run", self.run)
        for f in self.files:
            self.touch(f.name)

    def touch(self, name):
        self.clock += 10
        for f in self.files:
            if f.name == name:
                os.utime(f, (self.clock, self.clock))

    def run(self, cmd, name, verbose):
        self.ran.append(name)
        if name in self.failing:
            raise RuntimeError(f"failed on {name}")
        target = cmd[cmd.index("-o") + 1]
        self.clock += 10
        with open(target, "w") as f:
            f.write(str(self.clock))
        os.utime(target, (self.clock, self.clock))

    def build(self):
        """What was compiled and linked, or the error."""
        self.ran = []
        build.build(jobs=1)
        return set(self.ran)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    return Tree(tmp_path, monkeypatch)


EVERY = {"one.cu", "two.cu", "torch_binding.cpp", "library.so", "binding.so"}


def test_what_changed_is_built_again_and_nothing_else(tree):
    assert not build.up_to_date() and tree.build() == EVERY
    assert build.up_to_date() and tree.build() == set()
    tree.touch("two.cu")
    assert not build.up_to_date() and tree.build() == {"two.cu", "library.so"}
    tree.touch("torch_binding.cpp")
    assert tree.build() == {"torch_binding.cpp", "binding.so"}
    tree.touch("args.h")
    assert tree.build() == EVERY
    assert build.up_to_date()


@pytest.mark.parametrize("failing", ["one.cu", "two.cu", "torch_binding.cpp", "library.so", "binding.so"])
@pytest.mark.parametrize("changed", ["args.h", "all.cuh"])
def test_a_build_after_one_that_failed_links_all_that_was_compiled(tree, changed, failing):
    tree.build()
    tree.touch(changed)
    since = tree.clock
    tree.failing = {failing}
    with pytest.raises(RuntimeError, match=failing):
        tree.build()
    assert not build.up_to_date()
    tree.failing = set()
    tree.build()
    assert build.up_to_date()
    for out in (build.OUT, build.BINDING_OUT):  # written after the change, not marked as new
        assert int(open(out).read()) > since


def test_another_torch_needs_another_binding(tree, monkeypatch):
    tree.build()
    monkeypatch.setattr(build, "_installed", lambda: "another torch")
    assert not build.up_to_date()
    tree.failing = {"binding.so"}
    with pytest.raises(RuntimeError):
        tree.build()
    assert not build.up_to_date()  # the module of the torch before is still there
    tree.failing = set()
    assert tree.build() == {"torch_binding.cpp", "binding.so"}
    assert build.up_to_date() and tree.build() == set()
    os.remove(build.BINDING_FOR)
    assert not build.up_to_date() and tree.build() == {"torch_binding.cpp", "binding.so"}
