"""An engine whose KV pool is in 8 bits, on the GPU: logits and choices against the fp32 engine on the CPU that rounds the
rows it stores to the same codes (see kv8_cases for the tolerance), through decode graphs and without."""

import pytest
import torch

from kv8_cases import ENGINE_TOL, round_cache_rows
from minisgl.core import SamplingParams
from minisgl.kvcache.kv8_pool import KV8_DTYPES
from minisgl.models.synthetic import make_checkpoint
from test_engine_gpu import _check_against_oracle, _prompts, _run

pytestmark = pytest.mark.gpu

# Steps of 96 that may leave the tolerance in a model with experts: where two router logits are closer than the error of the
# hidden state another expert is taken, whatever computes the attention. The plain forms alone (bf16 against fp32 on the CPU, over
# the same cache) leave it in 4, 2 and 5 steps (int8) and 1, 4 and 1 (e4m3) with prompts of seeds 3, 4 and 5: a count of mean 3,
# which passes 12 once in 10^5 runs. A window or sinks that do not reach the operator move every step.
MOE_OUTLIERS = 12


@pytest.mark.parametrize("graphs", [0, 16])
@pytest.mark.parametrize("name", list(KV8_DTYPES))
@pytest.mark.parametrize("preset", ["tiny-qwen3", "tiny-llama", "tiny-gpt-oss"])
def test_engine_tracks_rounded_rows(tmp_path, preset, name, graphs, free_port, monkeypatch):
    """Chunked prompts, prefixes that are found in the cache, decoding; for MoE models steps whose experts are chosen
    otherwise may leave the tolerance."""
    path = make_checkpoint(preset, str(tmp_path / preset), dtype=torch.bfloat16)
    prompts = _prompts(11, 1024, seed=3)
    prompts.append(prompts[0][:16] + prompts[1])
    sp = SamplingParams(max_tokens=8, ignore_eos=True)
    outs, rows = _run(path, prompts, sp, free_port, tap=True, dtype=torch.bfloat16, max_running_req=32, num_page_override=1024,
                      page_size=16 if graphs else 64, cuda_graph_max_bs=graphs, max_extend_tokens=100, kv_cache_dtype=name)
    rows = [rows[i][-len(o):] for i, o in enumerate(outs)]  # (a prompt's earlier chunks give rows too)
    round_cache_rows(monkeypatch, name)
    _check_against_oracle(path, prompts, outs, free_port + 1, tol=ENGINE_TOL[name], gpu_rows=rows,
                          outliers=MOE_OUTLIERS if preset == "tiny-gpt-oss" else 0)
