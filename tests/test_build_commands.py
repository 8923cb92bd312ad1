"""The commands that build the operators' module for torch."""
import os

from mplayers_amd import _build


def test_the_module_for_torch_is_built_with_warnings_and_the_compilers_headers(tmp_path, monkeypatch):
  command = _build._autograd_command()
  assert "-w" not in command and {"-Wall", "-Wextra"} <= set(command)
  # headers beside the compiler that is named, by path or found on PATH
  root = tmp_path / "rocm"
  for name in ("bin/hipcc", "include/hip/hip_runtime.h"):
    (root / name).parent.mkdir(parents=True, exist_ok=True)
    (root / name).write_text("")
  (root / "bin/hipcc").chmod(0o755)
  include = os.path.realpath(root / "include")
  monkeypatch.setenv("HIPCC", str(root / "bin/hipcc"))
  assert include in _build._autograd_command()
  monkeypatch.setenv("HIPCC", "hipcc")
  monkeypatch.setenv("PATH", str(root / "bin") + os.pathsep + os.environ["PATH"])
  assert include in _build._autograd_command()
  # a compiler without headers beside it
  (root / "include/hip/hip_runtime.h").unlink()
  assert "/opt/rocm/include" in _build._autograd_command()
