"""The decode benchmark's arguments reach the decoder."""
import importlib.util
import os
import sys
import types

import pytest


@pytest.mark.parametrize("bits", [None, 8, 16])
def test_cache_bits_reach_the_decoder(bits, monkeypatch):
    import mesh_b200.models.e2b as e2b
    import mesh_b200.utils.status as status
    import mesh_b200.distributed as distributed
    seen = {}
    ctx = types.SimpleNamespace(rank=0, world=1)
    monkeypatch.setitem(sys.modules, "common", types.SimpleNamespace(emit=lambda *a: None, init=lambda: ctx))
    monkeypatch.setattr(e2b, "bench_decode", lambda c, **kw: seen.update(kw) or {})
    monkeypatch.setattr(status, "check_status", lambda *a: None)
    monkeypatch.setattr(distributed, "shutdown", lambda: None)
    monkeypatch.setattr(sys, "argv", ["decode.py", "--steps", "5", "--prompt", "7"] + ([] if bits is None else ["--cache-bits", str(bits)]))
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "benchmarks", "decode.py")
    spec = importlib.util.spec_from_file_location("bench_decode_script", path)
    script = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(script)
    script.main()
    assert seen == dict(steps=5, prompt_len=7, cache_bits=bits or 16)
