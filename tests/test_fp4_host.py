"""Host side of the 4-bit MLPs in the engine (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from glm53.engine.backend import GPUBackend
from glm53.ops import _ext


def backend(mlp4):
    b = GPUBackend.__new__(GPUBackend)
    b.sampler, b.rt, b.mlp4 = (lambda lg: lg.argmax(-1)), SimpleNamespace(px=None), mlp4
    return b


def test_argmax_raises_when_a_wait_of_the_4bit_kernels_ran_out(monkeypatch):
    words = [0, 0x6b40]
    asked = []
    monkeypatch.setattr(_ext, "require", lambda: SimpleNamespace(fp4_error=lambda d: asked.append(d) or words.pop(0)))
    logits = SimpleNamespace(device=torch.device("cuda", 3), argmax=lambda dim: torch.tensor([5]))
    assert backend(True).argmax(logits) == [5]
    with pytest.raises(RuntimeError, match="bounded wait ran out .code 0x6b40"):
        backend(True).argmax(logits)
    assert asked == [3, 3]


def test_argmax_does_not_ask_without_4bit_mlps(monkeypatch):
    monkeypatch.setattr(_ext, "require", lambda: pytest.fail("asked"))
    assert backend(False).argmax(torch.eye(3)) == [0, 1, 2]


def test_option_order_of_positional_callers():
    """The 4-bit options stand behind the ones that were there: sp_mla keeps its place."""
    import dataclasses

    from glm53.api.offline import LLMOptions
    names = [f.name for f in dataclasses.fields(LLMOptions)]
    assert names[names.index("ep") + 1] == "sp_mla" and names[-2:] == ["mlp4", "mlp4_act4"]


def test_act4_alone_is_refused():
    from glm53.api.offline import LLMOptions
    from glm53.api.server import build_parser, options_from_args
    with pytest.raises(ValueError, match="mlp4_act4 .* needs mlp4"):
        LLMOptions(mlp4_act4=True)
    with pytest.raises(ValueError, match="mlp4_act4 .* needs mlp4"):
        options_from_args(build_parser().parse_args(["--mlp4-act4"]))
    assert LLMOptions(mlp4="mxfp4", mlp4_act4=True).mlp4_act4
