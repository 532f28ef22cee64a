"""The stream that an operator is given is one of its tensors' device, whatever device is current (CPU only: torch's
stream calls are recorded)."""
from __future__ import annotations

from contextlib import nullcontext
from types import SimpleNamespace

import pytest
import torch

from stagehand_amd import int8, qk_norm


@pytest.fixture
def made(monkeypatch):
    """Streams that are made, then the one that becomes current."""
    calls = []

    def stream(kind):
        def make(*args):
            calls.append((kind, *args))
            return SimpleNamespace(device=args[-1])
        return make

    monkeypatch.setattr(torch.cuda, "ExternalStream", stream("external"))
    monkeypatch.setattr(torch.cuda, "default_stream", stream("default"))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: calls.append(("current", s.device)) or nullcontext())
    return calls


ON = torch.device("cuda", 1)
TENSOR = SimpleNamespace(is_cuda=True, device=ON, qweight=SimpleNamespace(is_cuda=True, device=ON))


class Reached(Exception):
    pass


CALLS = [
    (int8, "quantize_tokens", lambda f, s: f(TENSOR, stream=s)),
    (int8, "matmul_i8", lambda f, s: f(None, TENSOR, stream=s)),
    (int8, "linear_i8", lambda f, s: f(None, TENSOR, stream=s)),
    (qk_norm, "qk_norm_rope", lambda f, s: f(TENSOR, None, stream=s)),
]


@pytest.mark.parametrize("module,name,call", CALLS, ids=[c[1] for c in CALLS])
def test_a_stream_is_taken_on_the_tensors_device(monkeypatch, made, module, name, call):
    operator = getattr(module, name)

    def inner(*args, **kw):  # the call on the current stream
        assert kw.get("stream") is None
        raise Reached

    monkeypatch.setattr(module, name, inner)
    for given, want in ((77, [("external", 77, ON), ("current", ON)]), (0, [("default", ON), ("current", ON)]),
                        (SimpleNamespace(device=ON), [("current", ON)])):
        made.clear()
        with pytest.raises(Reached):
            call(operator, given)
        assert made == want
    made.clear()
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        call(operator, SimpleNamespace(device=torch.device("cuda", 0)))
    assert made == []


def test_a_stream_for_host_tensors_is_refused(made):
    x = torch.zeros(2, 8)
    for call in (lambda: int8.quantize_tokens(x, stream=5), lambda: qk_norm.qk_norm_rope(x[None, None], None, stream=5)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    assert made == []
