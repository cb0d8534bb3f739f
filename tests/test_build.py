"""The extension's build: a changed header reaches every object."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHOW = ("from distutils.core import run_setup\n"
        "(e,) = run_setup('setup.py', stop_after='init').ext_modules\n"
        "print('RESULT', sorted(e.depends), e.extra_compile_args['nvcc'])\n")


def extension(folder):
    run = subprocess.run([sys.executable, "-c", "import setuptools\n" + SHOW], cwd=folder,
                         capture_output=True, text=True, check=True)
    return next(line for line in run.stdout.splitlines() if line.startswith("RESULT"))


def test_headers_are_dependencies(tmp_path):
    """The build tool compares commands, since HIP sources get no dependency files."""
    source = tmp_path / "deepreduce_amd" / "ops" / "src"
    shutil.copytree(os.path.join(ROOT, "deepreduce_amd", "ops", "src"), source)
    shutil.copy(os.path.join(ROOT, "setup.py"), tmp_path)
    before = extension(tmp_path)
    assert "lm_ops.h" in before and extension(tmp_path) == before
    with open(source / "lm_ops.h", "a") as f:
        f.write("// changed\n")
    assert extension(tmp_path) != before
