"""The tiny proxy on the GPU runtime against the fp32 CPU oracle: teacher-forced logits over a
128-token prompt + greedy continuation, verify windows with partial commit (KDA state rollback), and the DSA
sparse path (context past index_topk = 64)."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _dev_weights(w):
    from tests.test_gpu_kernels import _to_dev
    return _to_dev(w)


def _oracle(cfg, weights, n_prompt=128, n_gen=24):
    from glm53.models.reference import ReferenceModel
    m = ReferenceModel(weights)
    g = torch.Generator().manual_seed(0)
    prompt = torch.randint(0, cfg.vocab, (n_prompt,), generator=g).tolist()
    toks, logits = m.generate_greedy(prompt, n_gen)
    return prompt, toks, torch.stack(logits)


@pytest.fixture(scope="module")
def oracle_run(tiny_cfg, tiny_weights):
    return _oracle(tiny_cfg, tiny_weights)


@pytest.fixture(scope="module")
def dense_setup(tiny_ckpt):
    """The tiny proxy with index_topk 256: every query of a 152-token run sees all keys (no discrete selection)."""
    import glm53
    from glm53.models import weights as W
    cfg = dataclasses.replace(glm53.tiny_config(), index_topk=256)
    w = W.prepare(W.DictSource(tiny_ckpt), cfg)
    return cfg, w, _oracle(cfg, w)


def _close(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    cos = torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0).item()
    return cos, (a - b).abs().max().item()


def _runtime(weights):
    from glm53.models.runtime import Runtime, RuntimeConfig
    return Runtime(_dev_weights(weights), RuntimeConfig(max_rows=64, kv_slots=1024, block_size=64, max_blocks=16))


def _run_teacher_forced(weights, oracle):
    from glm53.models.session import Sequence
    prompt, toks, ref_logits = oracle
    seq = Sequence(_runtime(weights))
    lg = seq.prefill(prompt, chunk=64)
    coss = [_close(lg[0], ref_logits[0])[0]]
    agree = 0
    for i, t in enumerate(toks[:-1]):
        lg = seq.verify([t])
        seq.commit(1)
        coss.append(_close(lg[0], ref_logits[i + 1])[0])
        agree += int(torch.argmax(lg[0]).item() == toks[i + 1])
    return torch.tensor(coss), agree


def test_tiny_model_dense_context_tight(dense_setup):
    # discrete near-ties remain even with dense attention: the MoE top-k can pick a different expert when a bf16
    # rounding difference moves a router logit across the k-th/k+1-th boundary; such steps are rare
    cfg, w, oracle = dense_setup
    coss, agree = _run_teacher_forced(w, oracle)
    assert (coss > 0.999).float().mean() >= 0.8 and coss.min() > 0.95, coss
    assert agree >= len(oracle[1]) - 4


@pytest.mark.w8a8
def test_tiny_model_dense_context_w8a8_prefill(dense_setup):
    """The default prefill policy (per-row e4m3 activations for the KDA input and MLA output projections, the
    reference's production choice) stays close to the fp32 oracle; decode rows are exact W8A16 either way."""
    from glm53.ops import kernels as K
    assert {"kda_in_proj", "mla_o_proj"} <= K.W8A8_PROJ or K.PREFILL_W8A8 or not K.W8A8_PROJ
    cfg, w, oracle = dense_setup
    coss, agree = _run_teacher_forced(w, oracle)
    assert coss.min() > 0.95 and (coss > 0.99).float().mean() >= 0.9, coss
    assert agree >= len(oracle[1]) - 4


def test_tiny_model_sparse_dsa(tiny_weights, oracle_run):
    # past index_topk a bf16/fp8 rounding difference can flip a near-tied DSA pool choice (a discrete change of a
    # few attended keys), which moves single steps; the bulk of the steps must still agree tightly
    coss, agree = _run_teacher_forced(tiny_weights, oracle_run)
    assert coss.median() > 0.9995 and coss.min() > 0.95, coss
    assert agree >= len(oracle_run[1]) - 5


def test_tiny_model_verify_window_and_rollback(dense_setup):
    """A window of 8 rows gives each row's logits; keeping 3 of them rolls the KDA state back so that the
    continuation matches the oracle."""
    from glm53.models.session import Sequence
    cfg, w, (prompt, toks, ref_logits) = dense_setup
    seq = Sequence(_runtime(w))
    seq.prefill(prompt, chunk=64)
    window = [toks[0], toks[1], toks[2], 7, 8, 9, 10, 11]       # 3 correct drafts, then garbage
    lg = seq.verify(window)
    coss = [_close(lg[i], ref_logits[i + 1])[0] for i in range(3)]
    seq.commit(3)
    for i in range(3, 10):
        lg = seq.verify([toks[i]])
        seq.commit(1)
        coss.append(_close(lg[0], ref_logits[i + 1])[0])
    coss = torch.tensor(coss)
    assert (coss > 0.9995).float().mean() >= 0.8 and coss.min() > 0.95, coss


def test_tiny_model_chunked_prefill_matches_stepwise(dense_setup):
    """A 128-token prefill in 64-row chunks (chunked KDA kernel) gives the same last-token logits as 128 single
    steps (recurrent kernel)."""
    from glm53.models.session import Sequence
    cfg, w, (prompt, toks, ref_logits) = dense_setup
    rt = _runtime(w)
    seq = Sequence(rt)
    a = seq.prefill(prompt, chunk=64)[0].clone()
    seq.reset()
    for t in prompt:
        b = seq.verify([t])
        seq.commit(1)
    cos, mx = _close(a, b[0])
    assert cos > 0.9995, (cos, mx)


class _Dequantised:
    """Dense weights where the oracle reads the codes and row scales of a Linear8."""

    def __init__(self, w):
        self.w, self.dense, self.s = self, w.float().cpu(), torch.ones(w.shape[0])

    def view(self, dtype):
        return self.dense


def _oracle_mlp4(w, ckpt, fmt):
    """The fp32 oracle's weights with every dense MLP replaced by the values of its 4-bit form."""
    import copy
    from glm53.models import weights as W
    from glm53.ops import fp4

    def values(t):
        return fp4.dequantize4(fp4.quantize4(t.to(torch.bfloat16).to(DEV), fmt), torch.float32).cpu()

    w = copy.copy(w)
    w.layers = [copy.copy(lw) for lw in w.layers]
    for lw in w.layers:
        p = f"model.layers.{lw.index}.mlp."
        gate, up, down = (values(ckpt[p + n + "_proj.weight"]) for n in ("gate", "up", "down"))
        lw.mlp = W.MLPW(_Dequantised(torch.cat([gate, up])), _Dequantised(down), gate.shape[0])
    return w


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_tiny_model_mlp4(fmt):
    """Dense MLPs in 4 bits in every layer (no expert choice that a rounding could flip): prefill in 64-row chunks and greedy
    decode against the oracle with the same 4-bit values."""
    import glm53
    from glm53.models import weights as W
    from glm53.models.runtime import Runtime, RuntimeConfig
    from glm53.models.session import Sequence
    cfg = dataclasses.replace(glm53.tiny_config(), index_topk=256, mlp_kinds=["dense"] * 4)
    ckpt = W.random_checkpoint(cfg, seed=0)
    w4 = W.prepare(W.DictSource(ckpt), cfg, device=DEV, mlp4=fmt)
    assert w4.layers[0].mlp.gu is None and w4.layers[0].mlp.four.gu.fmt == fmt
    w8 = W.prepare(W.DictSource(ckpt), cfg)
    assert w4.nbytes() < w8.nbytes()
    prompt, toks, ref_logits = _oracle(cfg, _oracle_mlp4(w8, ckpt, fmt))
    for act4 in (False, True):
        rt = Runtime(w4, RuntimeConfig(max_rows=64, kv_slots=1024, block_size=64, max_blocks=16, mlp4_act4=act4))
        seq = Sequence(rt)
        lg = seq.prefill(prompt, chunk=64)
        coss = [_close(lg[0], ref_logits[0])[0]]
        for i, t in enumerate(toks[:-1]):
            lg = seq.verify([t])
            seq.commit(1)
            coss.append(_close(lg[0], ref_logits[i + 1])[0])
        # act4: the prompt's MLP activations are quantised, and with them the state that decoding starts from
        assert min(coss) > (0.95 if act4 else 0.999), (act4, coss)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 8, 40])
def test_shared_expert_mlp4(tiny_ckpt, tiny_cfg, fmt, rows):
    """A MoE layer whose shared expert is in 4 bits: the routed sum of an fp8 run plus the block in 64 bits, on the side
    stream (decode windows) and after the routed experts."""
    from glm53.models import weights as W
    from glm53.models.runtime import Runtime, RuntimeConfig
    from glm53.ops import fp4
    rc = RuntimeConfig(max_rows=48, kv_slots=256, max_blocks=4)
    w4 = W.prepare(W.DictSource(tiny_ckpt), tiny_cfg, device=DEV, mlp4=fmt)
    w8 = W.prepare(W.DictSource(tiny_ckpt), tiny_cfg, device=DEV)
    lw4, lw8 = w4.layers[1], w8.layers[1]
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, tiny_cfg.hidden, generator=g, device=DEV).to(torch.bfloat16)
    p = "model.layers.1.mlp.shared_experts."
    gate, up, down = (fp4.dequantize4(fp4.quantize4(tiny_ckpt[p + n + "_proj.weight"].to(DEV).to(torch.bfloat16), fmt),
                                      torch.float32).double() for n in ("gate", "up", "down"))
    lim = tiny_cfg.limit
    gv, uv = (x.double() @ gate.t()).clamp(max=lim), (x.double() @ up.t()).clamp(-lim, lim)
    h = (gv * torch.sigmoid(gv) * uv).to(torch.bfloat16).double()
    ref = h @ down.t()
    outs = {}
    for name, w, lw in (("4", w4, lw4), ("8", w8, lw8)):
        for overlap in (True, False):
            rt = Runtime(w, rc)
            rt.overlap = rt.overlap and overlap
            rt._keep_window, rt._sp, rt._fused = True, None, False
            rt.normed[:rows] = x
            rt._moe(lw, rows)
            torch.cuda.synchronize()
            outs[name, overlap] = rt.branch[:rows].double()
    m = w8.layers[1].moe.shared
    g8 = x.double() @ (m.gu.w.view(torch.float8_e4m3fn).double() * m.gu.s.double()[:, None]).t()
    n = m.width
    rb = lambda t: t.to(torch.bfloat16).double()                                  # noqa: E731
    gv, uv = rb(g8[:, :n]).clamp(max=lim), rb(g8[:, n:]).clamp(-lim, lim)
    ref8 = rb(gv * torch.sigmoid(gv) * uv) @ (m.down.w.view(torch.float8_e4m3fn).double() * m.down.s.double()[:, None]).t()
    routed = outs["8", False] - ref8
    # h (and, in the fp8 run, gate and up) may round to bf16 on either side: half a step each, 2^-8 of the magnitudes
    tol = 2.0 ** -8 * (h.abs() @ down.abs().t()) + 3 * 2.0 ** -8 * (rb(gv * torch.sigmoid(gv) * uv).abs() @ (
        m.down.w.view(torch.float8_e4m3fn).double().abs() * m.down.s.double()[:, None]).t()) + 1e-5 * outs["8", False].abs()
    for overlap in (True, False):
        assert ((outs["4", overlap] - (routed + ref)).abs() <= tol).all()


def test_engine_with_mlp4_graphs():
    """The engine (CUDA graphs, speculation, side stream) on 4-bit MLPs: the tokens of a run without graphs."""
    from glm53.api.offline import LLM, LLMOptions
    from glm53.engine.llm import SamplingParams
    outs = []
    for graphs in (True, False):
        llm = LLM(LLMOptions(model="tiny", max_seqs=2, max_model_len=512, prefill_chunk=128, mlp4="nvfp4", mlp4_act4=True,
                             cuda_graphs=graphs, k_fixed=4))
        outs.append([o["token_ids"] for o in llm.generate([[1, 2, 3] * 50, [9, 8, 7] * 20],
                                                          SamplingParams(max_tokens=24))])
    assert outs[0] == outs[1]
