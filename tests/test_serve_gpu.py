"""The serving example: pages, cache rows, prompt attention and draft trees together.

Its check compares two bf16 computations of one value. Either rounds keys, values, queries
and latent outputs to bf16 on its way (at most five roundings of 2^-8 each, of values that
the outputs are weighted means and 512-term sums of): 5 * 2^-8 of the outputs' size for a
typical element; the largest of some ten thousand is within five times that."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("requests,heads,prompt,drafts", [(3, 8, 150, 5), (2, 128, 70, 3), (1, 20, 1, 12)])
def test_forms_agree(requests, heads, prompt, drafts):
    import importlib.util

    spec = importlib.util.spec_from_file_location("serve", os.path.join(ROOT, "ada-mla_b200", "serve.py"))
    serve = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(serve)
    import ada_mla

    assert serve.run(requests, heads, prompt, drafts) <= 25 * 2.0 ** -8
    assert ada_mla.mla_get_device_error() == 0


def test_command():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "ada-mla_b200", "serve.py"), "--requests", "2", "--heads", "8", "--prompt", "90"],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert "differ by" in out.stdout
