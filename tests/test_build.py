"""CPU tests of the build script and of what links against its libraries."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

REPO = Path(__file__).resolve().parents[1]


def test_builds_without_torch(built):
    """Everything but the torch extension is built where torch is missing."""
    code = """
import sys
sys.modules["torch"] = None
import build
commands = []
build._stale = lambda target, inputs: True
build._run = lambda command, verbose: commands.append(command)
outputs = build.build()
targets = {command[command.index("-o") + 1].rsplit("/", 1)[-1] for command in commands}
assert {"liblrrt.so", "liblrrt_ops.so", "liblrrt_qwen.so", "paged_ops.cubin"} <= targets, targets
assert "lrrt_ops_torch.so" not in targets and "ops_torch" not in outputs
"""
    result = subprocess.run([sys.executable, "-c", code], cwd=REPO / "light-rocm-runtime_b200",
                            capture_output=True, text=True, timeout=120)
    assert result.returncode == 0, result.stderr
    assert "torch is not installed" in result.stdout


def test_a_program_links_the_driver_alone(built, tmp_path):
    """A program that names liblrrt_qwen and liblrrt, as before the operators'
    library came between, links and starts."""
    source = tmp_path / "program.cpp"
    source.write_text('#include "lrrt_qwen.h"\n'
                      "int main() { return lrq_last_error() == nullptr; }\n")
    library = built["driver"].parent
    program = tmp_path / "program"
    environment = {k: v for k, v in os.environ.items() if k != "LD_LIBRARY_PATH"}
    for command in ([shutil.which("g++"), f"-I{REPO / 'include'}", str(source), "-o",
                     str(program), f"-L{library}", "-llrrt_qwen", "-llrrt",
                     f"-Wl,-rpath,{library}"], [str(program)]):
        result = subprocess.run(command, capture_output=True, text=True, env=environment,
                                timeout=120)
        assert result.returncode == 0, result.stderr
