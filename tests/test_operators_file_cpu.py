"""perf/operators.py without a GPU: where its calls go."""
import importlib
import types

import torch


def test_calls_go_to_the_stream_that_is_current(pkg, monkeypatch):
    operators = importlib.import_module("perf.operators")
    made = []
    call = lambda *args, stream=None: made.append(stream)  # noqa: E731
    fake = types.SimpleNamespace(paged_attention=call, cache_write=call, cache_read=call, paged_cache=call, paged_batch=call, paged_attention_params=lambda *a, **k: None,
                                 paged_attention_workspace=lambda *a: 0)
    monkeypatch.setattr(operators, "importlib", types.SimpleNamespace(import_module=lambda name: fake))
    for op in ("attend", "write", "keep", "read"):
        state = dict(case=dict(op=op, q=1, kv=1, heads=1, d_h=16), tokens=1, k=types.SimpleNamespace(device=torch.device("cuda", 0)),
                     **{x: None for x in ("v", "q_start", "kv_len", "pages", "K", "V", "Q", "O", "K_out", "V_out")})
        for stream in (11, 12):
            monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: stream)
            made.clear()
            operators._through_package(state)
            sent = [s for s in made if s is not None]
            assert sent and set(sent) == {stream}, op
