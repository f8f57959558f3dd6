"""build_native.py: what is built where, and what is built again."""
import sys

import pytest

import __graft_entry__
import build_native


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """build() with its compiler and linker calls recorded, not run."""
    calls = []
    monkeypatch.setattr(build_native, "BUILD", tmp_path / "build")
    monkeypatch.setattr(build_native, "PKG", tmp_path)
    monkeypatch.setattr(build_native, "_run", lambda cmd: (calls.append(cmd), open(cmd[cmd.index("-o") + 1], "w").close()))
    return calls


def torch_at(monkeypatch, tmp_path, libs):
    where = tmp_path / "torch"
    (where / "lib").mkdir(parents=True)
    for lib in libs:
        (where / "lib" / lib).touch()
    monkeypatch.setattr(build_native, "torch_dir", lambda: where)


@pytest.mark.parametrize("libs", [None, (), ("libc10.so", "libtorch_cpu.so"), ("libc10.so", "libc10_cuda.so")])
def test_without_a_rocm_torch_everything_else_is_built(recorded, monkeypatch, tmp_path, libs):
    if libs is None:
        monkeypatch.setattr(build_native, "torch_dir", lambda: None)
    else:
        torch_at(monkeypatch, tmp_path, libs)
    out = build_native.build(jobs=1)
    assert "fp8" not in out and {"module", "kernels", "sentinel", "aqlpmc_plugin"} <= set(out)
    assert not any("fp8" in word for cmd in recorded for word in cmd)


def test_with_a_rocm_torch_the_operators_are_built(recorded, monkeypatch, tmp_path):
    torch_at(monkeypatch, tmp_path, ("libc10.so", "libc10_hip.so"))
    assert "fp8" in build_native.build(jobs=1)


def test_the_entry_does_not_want_what_was_not_built(monkeypatch):
    real = {"module": "m"}
    monkeypatch.setattr(build_native, "build", lambda **kw: dict(real))
    monkeypatch.setitem(sys.modules, "kubernetes_gpu_exporter_amd.ops.fp8", None)  # an import of it fails
    __graft_entry__.build()


def compiled(calls):
    """The sources compiled by the recorded calls, which are then forgotten."""
    out = {word.rsplit("/", 1)[1] for cmd in calls for word in cmd if "/csrc/" in word and word.endswith((".cc", ".hip"))}
    calls.clear()
    return out


def test_objects_of_another_command_are_built_again(recorded, monkeypatch, tmp_path):
    torch_at(monkeypatch, tmp_path, ("libc10_hip.so",))
    version = tmp_path / "torch" / "version.py"
    version.write_text("__version__ = '1'")
    build_native.build(jobs=1)
    everything = compiled(recorded)
    assert {"fp8_torch.cc", "gemm_bf16.hip", "sentinel_hsaco.hip", "engine.cc"} <= everything
    build_native.build(jobs=1)
    assert not compiled(recorded)
    version.write_text("__version__ = '2'")
    build_native.build(jobs=1)
    assert compiled(recorded) == {"fp8_torch.cc"}
    monkeypatch.setattr(build_native, "HIP_FLAGS", ["-another"])
    build_native.build(jobs=1)
    assert compiled(recorded) == {name for name in everything if name.endswith(".hip")}
    build_native.build(jobs=1, sanitize="undefined")
    assert compiled(recorded) == everything - {"sentinel_hsaco.hip", "calib_hsaco.hip"}
    build_native.build(jobs=1, force=True)
    assert compiled(recorded) == everything


def test_an_object_whose_compiler_failed_is_built_again(recorded, monkeypatch):
    build_native.build(jobs=1)
    compiled(recorded)
    run = build_native._run

    def fails(cmd):
        run(cmd)
        raise RuntimeError("failed")
    monkeypatch.setattr(build_native, "_run", fails)
    with pytest.raises(RuntimeError):
        build_native.build(jobs=1, force=True)
    monkeypatch.setattr(build_native, "_run", run)
    first = compiled(recorded)
    build_native.build(jobs=1)
    assert first & compiled(recorded)
