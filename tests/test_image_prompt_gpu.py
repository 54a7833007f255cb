"""The example that runs the operators of language models together, behind a network of the framework."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_steps_over_the_cache_give_what_the_whole_sequence_gives(gpu_mode):
    path = os.path.join(ROOT, "mini-caffe_amd", "examples", "image_prompt.py")
    spec = importlib.util.spec_from_file_location("image_prompt", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    answers = example.main(steps=12)          # (asserts it)
    assert answers.shape == (2, 12) and len(set(answers.flatten().tolist())) > 2
