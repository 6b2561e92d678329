"""qmlp.tokens.precompile leaves every kernel in the cache that calls with values of the type need (no device needed)."""
import os
import re
import subprocess
import sys

import pytest

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quick-mlp_amd")


@pytest.mark.parametrize("dtype,name", [("bfloat16", "__bf16")])
def test_layer_norms_with_weights_in_single_precision_are_compiled_too(dtype, name, tmp_path):
    """Rows of 16 bits with float weights: what FusedLayerNorm has unless it is told otherwise."""
    program = "import torch, qmlp; qmlp.set_kernel_cache_dir(%r); qmlp.tokens.precompile(torch.%s)" % (str(tmp_path), dtype)
    subprocess.run([sys.executable, "-c", program], check=True, timeout=600, env=dict(os.environ, PYTHONPATH=PACKAGE))
    kernels = set()
    for file in os.listdir(tmp_path):
        with open(tmp_path / file, "rb") as f:
            kernels.update(k.decode() for k in re.findall(rb"qmlp::kernel::([A-Za-z]+<[^<>]*>|[A-Za-z]+)", f.read(512)))
    own = [k for k in kernels if k.startswith("LayerNorm") and "<%s, %s" % (name, name) in k]
    assert len(own) == 22   # 10 shapes of rows and the one of long rows, forward and adjoint
    for k in own:
        assert k.replace("%s, %s" % (name, name), "%s, float" % name) in kernels, k
    assert {"LayerNormSumKernel<float>", "LayerNormSumKernel<%s>" % name, "LayerNormLongSumsKernel<%s>" % name} <= kernels
