"""Calls of the 4-bit operators that are refused before anything is launched (no GPU needed)."""
import pytest
import torch

from glm53.ops import fp4

BF = torch.bfloat16


def u8(n):
    return torch.zeros(n, dtype=torch.uint8)


@pytest.mark.parametrize("call,words", [
    (lambda: fp4.quantize4(torch.zeros(4, 64, dtype=BF)), "CUDA"),
    (lambda: fp4.quantize4(torch.zeros(4, 64, dtype=BF), "fp4"), "unknown 4-bit format"),
    (lambda: fp4.Matrix4.from_parts(u8(16384), u8(2048), torch.ones(3), 3, 24, "nvfp4"), r"multiple of 16, got \[3, 24\]"),
    (lambda: fp4.Matrix4.from_parts(u8(16384), u8(1024), None, 3, 48, "mxfp4"), r"multiple of 32, got \[3, 48\]"),
    (lambda: fp4.Matrix4.from_parts(u8(16384), u8(1024), None, 0, 64, "mxfp4"), r"rows >= 1"),
    (lambda: fp4.Matrix4.from_parts(u8(16384), u8(1024), None, 1 << 31, 64, "mxfp4"), r"at most"),
    (lambda: fp4.Matrix4.from_parts(u8(16384), u8(1024), None, 128, 256, "mxfp4"), "16384 contiguous"),
    (lambda: fp4.pack_mlp4(torch.zeros(48, 64), torch.zeros(48, 64), torch.zeros(64, 48)), "multiple of 32, got 48"),
    (lambda: fp4.pack_mlp4(torch.zeros(64, 64), torch.zeros(64, 32), torch.zeros(64, 64)), "one shape"),
    (lambda: fp4.pack_mlp4(torch.zeros(64, 64), torch.zeros(64, 64).to(BF), torch.zeros(64, 64)), "one shape"),
    (lambda: fp4.pack_mlp4(torch.zeros(64, 64), torch.zeros(64, 64), torch.zeros(64, 32)), r"down must be \[N, 64\]"),
])
def test_refused(call, words):
    with pytest.raises((RuntimeError, ValueError), match=words):
        call()


@pytest.mark.parametrize("kw,words", [
    (dict(mlp4="fp4"), "must be one of nvfp4, mxfp4"),
    (dict(mlp4="nvfp4", world=2), "world == 1"),
    (dict(mlp4="nvfp4"), "needs a CUDA device"),
])
def test_prepare_refuses(tiny_cfg, tiny_ckpt, kw, words):
    from glm53.models import weights as W
    with pytest.raises(ValueError, match=words):
        W.prepare(W.DictSource(tiny_ckpt), tiny_cfg, **kw)


def test_server_flags_reach_the_options():
    from glm53.api.server import build_parser, options_from_args
    o = options_from_args(build_parser().parse_args(["--mlp4", "mxfp4", "--mlp4-act4"]))
    assert o.mlp4 == "mxfp4" and o.mlp4_act4
    o = options_from_args(build_parser().parse_args([]))
    assert o.mlp4 is None and not o.mlp4_act4
