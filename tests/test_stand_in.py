"""The stand-in for the engine's contract has every name that the backend takes from it, and
smoke() and bench.py find the backend without the engine."""

import subprocess
import sys

import pytest

from conftest import ENGINE_INSTALLED, REPO
from baseline import stand_in


def test_it_has_the_contracts_names():
    import ast

    tree = ast.parse((REPO / "my_vllm_b200" / "contract.py").read_text())
    names = {alias.asname or alias.name for node in ast.walk(tree)
             if isinstance(node, ast.ImportFrom) and (node.module or "").startswith("nanovllm")
             for alias in node.names}
    assert names and all(hasattr(stand_in, name) for name in names)


@pytest.mark.skipif(ENGINE_INSTALLED, reason="the engine is installed")
def test_the_backend_is_found_without_the_engine():
    # in a process of its own: this one's modules are set up by the tests' configuration
    code = ("import bench\nfrom my_vllm_b200 import B200PagedBackend\n"
            "from my_vllm_b200 import contract\nassert not contract.ENGINE_CONTRACT\n"
            "import torch\nb = B200PagedBackend(8, 2, 128, 16, torch.bfloat16)\n"
            "assert bench.STAND_IN and b.num_q_heads == 8\n"
            "import importlib.util\nassert importlib.util.find_spec('nanovllm') is None\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr


@pytest.mark.skipif(ENGINE_INSTALLED, reason="the engine is installed")
def test_without_either_the_backend_says_what_is_missing():
    code = "import my_vllm_b200\nmy_vllm_b200.B200PagedBackend\n"
    run = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True)
    assert run.returncode != 0 and "nanovllm" in run.stderr
