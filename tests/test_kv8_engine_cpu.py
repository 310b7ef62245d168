"""An engine whose KV pool is in 8 bits, on the CPU: its logits against an fp32 engine that rounds the rows it stores to the
same codes, its pool, its options."""

import pytest
import torch

from kv8_cases import ENGINE_TOL, FMTS, nearest, round_cache_rows
from minisgl.core import SamplingParams
from minisgl.kvcache.kv8_pool import KV8_DTYPES, KV8Pool
from minisgl.models.synthetic import make_checkpoint
from test_engine_gpu import _check_against_oracle, _prompts, _run

KW = dict(dtype=torch.bfloat16, device="cpu", max_running_req=16)


@pytest.mark.parametrize("name", list(KV8_DTYPES))
@pytest.mark.parametrize("preset", ["tiny-qwen3", "tiny-llama", "tiny-qwen2"])
def test_engine_tracks_rounded_rows(tmp_path, preset, name, free_port, monkeypatch):
    """Chunked prompts, prefixes that are found in the cache, decoding."""
    path = make_checkpoint(preset, str(tmp_path / preset), dtype=torch.bfloat16)
    prompts = _prompts(5, 1024)
    prompts.append(prompts[0][:16] + prompts[1])
    sp = SamplingParams(max_tokens=5, ignore_eos=True)
    outs, rows = _run(path, prompts, sp, free_port, tap=True, kv_cache_dtype=name, page_size=16, max_extend_tokens=48, **KW)
    rows = [rows[i][-len(o):] for i, o in enumerate(outs)]  # (a prompt's earlier chunks give rows too)
    round_cache_rows(monkeypatch, name)
    _check_against_oracle(path, prompts, outs, free_port + 1, tol=ENGINE_TOL[name], gpu_rows=rows)


def test_windows_and_sinks(tmp_path, free_port, monkeypatch):
    """Alternating windows and sinks reach the operator; steps whose experts are chosen otherwise may leave the tolerance."""
    path = make_checkpoint("tiny-gpt-oss", str(tmp_path / "m"), dtype=torch.bfloat16)
    prompts = _prompts(6, 1024, seed=2)
    sp = SamplingParams(max_tokens=5, ignore_eos=True)
    outs, rows = _run(path, prompts, sp, free_port, tap=True, kv_cache_dtype="int8", page_size=16, **KW)
    round_cache_rows(monkeypatch, "int8")
    _check_against_oracle(path, prompts, outs, free_port + 1, tol=ENGINE_TOL["int8"], gpu_rows=rows, outliers=3)


@pytest.mark.parametrize("dtype", FMTS)
def test_pool(dtype):
    from minisgl.parallel.info import reset_tp_info
    from minisgl.parallel import set_tp_info

    reset_tp_info()
    set_tp_info(0, 1)
    try:
        pool = KV8Pool(2, 3, 64, 4, 16, dtype, torch.device("cpu"))
    finally:
        reset_tp_info()
    assert (pool.num_layers, pool.dtype, pool.device.type, pool.num_slots) == (3, dtype, "cpu", 64)
    assert pool.bytes_per_token * 64 == sum(pool.layer(i).nbytes() for i in range(3))
    k, v = torch.randn(2, 5, 2 * 64).to(torch.bfloat16)
    loc = torch.tensor([3, 60, 9, -1, 0], dtype=torch.int32)
    pool.store_kv(k, v, loc, 1)
    for x, got in zip((k, v), pool.load_kv(loc, 1)):
        codes, scale = nearest(x.view(5, 2, 64), dtype)
        want = (codes * scale).to(torch.bfloat16).float()
        want[3] = 0
        assert ((got.float() - want).abs() <= want.abs() * 2.0**-7).all()  # (one bf16 step where fp32 rounds to a tie)
    for i in (0, 2):
        assert not pool.layer(i).k_scale.any() and not pool.k_cache(i).view(torch.uint8).any()
    assert pool.v_cache(1) is pool.layer(1).v


@pytest.mark.parametrize("kw,match", [
    (dict(kv_cache_dtype="int4"), "auto"),
    (dict(kv_cache_dtype="int8", dtype=torch.float32), "bfloat16"),
])
def test_refused_options(tmp_path, kw, match, free_port):
    from minisgl.llm import LLM

    path = make_checkpoint("tiny-qwen3", str(tmp_path / "m"), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=match):
        LLM(path, distributed_port=free_port, **dict(KW, **kw))


def test_odd_pages_are_overridden(tmp_path, free_port):
    from minisgl.llm import LLM

    path = make_checkpoint("tiny-qwen3", str(tmp_path / "m"), dtype=torch.bfloat16)
    llm = LLM(path, distributed_port=free_port, kv_cache_dtype="int8", page_size=1, **KW)
    try:
        assert llm.engine.ctx.page_size == 64 and isinstance(llm.engine.kv_cache, KV8Pool)
    finally:
        llm.shutdown()


def test_command_line():
    from minisgl.server.args import build_parser, parse_args

    assert parse_args(["--model", "x", "--dtype", "bfloat16"]).kv_cache_dtype == "auto"
    assert parse_args(["--model", "x", "--dtype", "bfloat16", "--kv-cache-dtype", "fp8_e4m3"]).kv_cache_dtype == "fp8_e4m3"
    with pytest.raises(SystemExit):
        build_parser().parse_args(["--model", "x", "--kv-cache-dtype", "int4"])
