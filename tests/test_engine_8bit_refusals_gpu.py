"""What an engine with pages held in 8 bits refuses before it loads a model."""

from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_the_plain_attention_kernel_is_refused_at_once(model_dirs, tmp_path):
    from paged_llm_rs_amd import Engine, kernels
    from paged_llm_rs_amd.errors import ConfigError

    path = model_dirs("A", "float32")
    kernels.set_attention("tensor")
    try:
        with pytest.raises(ConfigError, match="attention tensor"):
            Engine(path, dtype="f32", cache_dtype="e4m3", num_blocks=8)
        Engine(path, dtype="f32", num_blocks=8)
    finally:
        kernels.set_attention("kernel")
    run = subprocess.run([sys.executable, str(ROOT / "bin" / "pagedllm"), "--model", str(path), "--prompt-ids", "1,2,3", "--cache-dtype", "e4m3", "--attention", "tensor"],
                         capture_output=True, text=True, timeout=100)
    assert run.returncode != 0 and "attention tensor" in run.stderr and "Traceback" not in run.stderr and "blocks of" not in run.stderr
