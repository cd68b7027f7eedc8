"""The build: the engine needs nvcc only; the tensor binding follows where it
can, and what is up to date is not built again."""

import subprocess

import pytest

from megakernels import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """An empty build folder, and compilers that write empty files. Returns the commands run."""
    csrc = tmp_path / "pkg" / "csrc"
    csrc.mkdir(parents=True)
    for name in ("ek_capi.cu", "ek_torch.cpp", "ek_host.h"):
        (csrc / name).write_text("")
    (csrc / "ek_prefix_attn.cu").write_text("int REGS = I8 ? 128 : 168;")
    for name, value in {"PKG_ROOT": tmp_path / "pkg", "CSRC": csrc, "OUT": tmp_path / "pkg" / "libek.so",
                        "BINDING": tmp_path / "pkg" / "_ekops.so"}.items():
        monkeypatch.setattr(b, name, value)
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        if "fail" in getattr(run, "on", ()) and any("ek_torch" in str(c) for c in cmd):
            raise subprocess.CalledProcessError(1, cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").write("")
        text = "".join(f"ptxas info    : Compiling entry function '_Z9many_rowsILi{d}ELb{i}EEvNS_10ManyParamsE' for 'sm_100a'\n"
                       f"ptxas info    : Used {r} registers, used 4 barriers\n" for d in (64, 128) for i, r in ((0, 168), (1, 128)))
        return subprocess.CompletedProcess(cmd, 0, stdout="", stderr=text)

    run.on = set()
    monkeypatch.setattr(b.subprocess, "run", run)
    commands.append(run.on)
    return commands


def compiled(commands, what):
    return [c for c in commands[1:] if any(what in str(x) for x in c)]


def test_everything_is_built_once(tree):
    assert b.build() == b.OUT and b.OUT.exists() and b.BINDING.exists()
    n = len(tree)
    b.build()
    assert len(tree) == n


def test_a_new_binding_source_leaves_the_engine_alone(tree):
    import os

    b.build()
    n, t = len(tree), b.OUT.stat().st_mtime
    os.utime(b.CSRC / "ek_torch.cpp", (t + 10, t + 10))
    b.build()
    assert len(tree) == n + 1 and compiled(tree[n - 1 :], "ek_torch.cpp")


@pytest.mark.parametrize("missing", ["g++", "torch", "CUDA"])
def test_the_engine_is_built_without_what_only_the_binding_needs(tree, monkeypatch, missing):
    import sys

    import torch

    if missing == "g++":
        monkeypatch.delenv("CXX", raising=False)
        which = b.shutil.which
        monkeypatch.setattr(b.shutil, "which", lambda n, *a, **k: None if n in ("g++", "c++") else which(n, *a, **k) or n)
    elif missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        monkeypatch.setattr(torch.version, "cuda", None)
    with pytest.warns(RuntimeWarning, match="_ekops.so is not built"):
        assert b.build() == b.OUT
    assert b.OUT.exists() and not b.BINDING.exists() and not compiled(tree, "ek_torch.cpp")
    n = len(tree)
    with pytest.warns(RuntimeWarning):
        b.build()
    assert len(tree) == n  # the engine is not built again


def test_a_binding_that_does_not_compile_is_an_error_after_the_engine(tree):
    tree[0].add("fail")
    with pytest.raises(subprocess.CalledProcessError):
        b.build()
    assert b.OUT.exists() and not b.BINDING.exists()


def test_registers_of_the_tensor_core_kernel_are_checked(tree, monkeypatch):
    """A compiler that allots others than the kernel's split of registers counts on fails the build."""
    text = "constexpr int REGS = I8 ? 128 : 168, SOFTMAX_REGS = 200;"
    (b.CSRC / "ek_prefix_attn.cu").write_text(text)
    b.build()
    assert any("-v" in c for c in compiled(tree, "ek_prefix_attn.cu"))
    (b.CSRC / "ek_prefix_attn.cu").write_text(text.replace("168", "160"))
    with pytest.raises(RuntimeError, match="many_rows.*168 registers.*160"):
        b.build(force=True)
    monkeypatch.setattr(b.subprocess, "run", lambda cmd, **kw: subprocess.CompletedProcess(cmd, 0, stdout="", stderr=""))
    with pytest.raises(RuntimeError, match="many_rows"):
        b.build(force=True)


def test_registers_of_the_source_as_it_is():
    """The numbers that the build compares with are found in the kernel's source."""
    assert b.expected_registers() == {0: 168, 1: 128}
