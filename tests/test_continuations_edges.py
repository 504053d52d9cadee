"""Drafted trees and beams without a GPU: which kernels a model's loading compiles."""
import pytest
import torch

from microllm_rocm_b200.config import get_architecture
from microllm_rocm_b200.engine import loading
from microllm_rocm_b200.kernels import ops
from microllm_rocm_b200.parts.base import Runtime
from microllm_rocm_b200.parts.build import build_model
from tests.helpers import tiny_config


@pytest.mark.parametrize("key, dtype, tensor_core", [("a", torch.float32, None), ("c", torch.float32, None), ("a", torch.bfloat16, None), ("c", torch.bfloat16, 64), ("d", torch.bfloat16, 128)])
def test_loading_compiles_what_draft_steps_and_beam_search_launch(key, dtype, tensor_core, monkeypatch):
    asked = []
    monkeypatch.setattr(loading.kernel_build, "compile_many", lambda items: asked.extend(items))
    loading.prepare_kernels(build_model(get_architecture("Qwen2ForCausalLM").build_spec(tiny_config(key)), Runtime(torch.device("cpu"), dtype)))
    want = [("drafts.cu", {}), ("cache_moves.cu", {}), ("beams.cu", {})] + ([("drafts_tc.cu", {"HEAD_DIM": tensor_core})] if tensor_core else [])
    assert all(asked.count(x) == 1 and x in ops.continuation_sources() for x in want)
    assert len([x for x in asked if x[0] == "drafts_tc.cu"]) == (1 if tensor_core else 0)
