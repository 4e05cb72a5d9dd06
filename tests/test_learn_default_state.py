"""Dropout's default random state starts from a seed of its own: with the samplers' seed, a mask's words would be
the words that chose neighbours and list entries under the same stream number."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_default_seed_is_not_the_samplers():
    code = ("import torch, gsampler_b200 as gs\n"
            "print(*torch.ops.gs_ops._CAPI_NextDropoutStream(), gs.Graph(4, 4)._CAPI_GetSeed())")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    seed, stream, graph_seed = map(int, out.stdout.split())
    assert stream == 0 and seed != graph_seed
    assert seed != 7777, "list sampling starts from it"
