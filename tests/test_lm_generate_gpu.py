"""A language model served: 4-bit projections, the token step and the choice
of the next token together, eager and captured."""

from __future__ import annotations

import pytest
import torch

from src.kernels.linear_w4 import dequantize_w4, quantize_w4
from src.kernels.logits import next_tokens
from src.models.inference import Mamba3Decoder
from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import Mamba3, MambaConfig, MambaLMHeadModel
from src.models.stack import Mamba3StackDecoder
from src.models.mamba3 import MambaBlock

pytestmark = pytest.mark.gpu

FUSED = dict(use_triton_full_fused=True)


def lm(seed=0, dtype=torch.float32, mlp=64, mimo=True, vocab=203, tie=False):
    torch.manual_seed(seed)
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=vocab, d_intermediate=mlp, tie_embeddings=tie,
                      ssm_cfg=dict(d_state=32, headdim=16, is_mimo=mimo, mimo_rank=4 if mimo else 1))
    return MambaLMHeadModel(cfg, device="cuda", dtype=dtype).eval()


def rounded(model, G):
    """The same model with every projection replaced by what its 4-bit form
    stands for."""
    import copy
    m = copy.deepcopy(model)
    with torch.no_grad():
        linears = [m.lm_head] + [lin for b in m.layers for lin in (b.mixer.in_proj, b.mixer.out_proj)]
        linears += [lin for f in (m.mlp_layers or []) for lin in (f.fc1, f.fc2)]
        for lin in linears:
            lin.weight.copy_(dequantize_w4(quantize_w4(lin.weight, G), lin.weight.dtype))
    return m


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("mimo,mlp", [(True, 64), (False, 0)])
@pytest.mark.parametrize("G", [32, 128])
def test_w4_decode_is_the_rounded_models(G, mimo, mlp, graph):
    model = lm(mimo=mimo, mlp=mlp)
    ids = torch.randint(0, 203, (3, 6), device="cuda")
    with torch.no_grad():
        want, _ = Mamba3LMDecoder(rounded(model, G), **FUSED).decode_sequence(ids)
        dec = Mamba3LMDecoder(model, use_cuda_graph=graph, w4_group_size=G, **FUSED)
        states = dec.init_state(3, device="cuda")
        if graph:
            dec.warmup_cuda_graph(states, n_warmup=0)
        got, _ = dec.decode_sequence(ids, states)
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)


def test_w4_layer_prefill_and_stack():
    torch.manual_seed(1)
    layer = Mamba3(64, d_state=32, headdim=16, is_mimo=True, mimo_rank=4, device="cuda")
    u = torch.randn(2, 9, 64, device="cuda")
    with torch.no_grad():
        dec = Mamba3Decoder(layer, w4_group_size=64, **FUSED)
        a, sa = dec.prefill(u, dec.init_state(2, device="cuda"))
        b, sb = dec.decode_sequence(u, dec.init_state(2, device="cuda"))
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
        for k in sa:
            torch.testing.assert_close(sa[k], sb[k], rtol=1e-4, atol=1e-4)
        blocks = [MambaBlock(64, dict(d_state=32, headdim=16, is_mimo=True, mimo_rank=4), device="cuda")
                  for _ in range(2)]
        st = Mamba3StackDecoder(blocks, w4_group_size=64, **FUSED)
        x, _ = st.step(u[:, 0].contiguous(), st.init_state(2, device="cuda"))
        assert x.shape == (2, 64) and bool(x.isfinite().all())


def test_w4_follows_a_changed_weight():
    """Eagerly after an in-place change, and in a captured step after the
    next look at the weight."""
    model = lm()
    ids = torch.randint(0, 203, (2,), device="cuda")
    with torch.no_grad():
        dec = Mamba3LMDecoder(model, use_cuda_graph=True, w4_group_size=64, **FUSED)
        states = dec.init_state(2, device="cuda")
        dec.warmup_cuda_graph(states, n_warmup=1)
        for st in states:
            for v in st.values():
                v.zero_()
        dec.step(ids, states)
        model.lm_head.weight.mul_(2.0)
        model.layers[0].mixer.in_proj.weight.mul_(0.5)
        fresh = Mamba3LMDecoder(model, w4_group_size=64, **FUSED)
        want, _ = fresh.step(ids, fresh.init_state(2, device="cuda"))
        eager, _ = Mamba3LMDecoder.step(_Eager(dec), ids, dec.init_state(2, device="cuda"))
        torch.testing.assert_close(eager, want, rtol=1e-5, atol=1e-5)
        for st in states:
            for v in st.values():
                v.zero_()
        got, _ = dec.step(ids, states)
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


class _Eager:
    """A captured decoder's eager step."""

    def __init__(self, dec):
        self._graph, self._step_eager = None, dec._step_eager


def by_hand(dec, row, new, kw):
    """One row, one token at a time, through the decoder's step."""
    vocab = dec.model.config.vocab_size
    toks, lps = list(row), []
    states = dec.init_state(1, device="cuda")
    for t in range(len(row) + new - 1):
        logits, states = dec.step(torch.tensor([toks[t]], device="cuda"), states)
        if t + 1 < len(row):
            continue
        h = torch.tensor([toks], device="cuda")
        ids, lp = next_tokens(logits[:, :vocab], h, None, torch.tensor([len(row)], device="cuda"), **kw(len(toks)))
        toks.append(int(ids)), lps.append(float(lp))
    return toks, lps


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("w4", [None, 32])
@pytest.mark.parametrize("sample", [False, True])
def test_generate_ragged_prompts(graph, w4, sample):
    model = lm(seed=3)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 203, (n,), generator=g).tolist() for n in (4, 1, 7)]
    L, new = 7, 6
    ids = torch.full((3, L), 9999, device="cuda")  # what lies behind a prompt is not read
    for b, p in enumerate(prompts):
        ids[b, :len(p)] = torch.tensor(p)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (7,), generator=g).int().cuda()
    kw = dict(repetition_penalty=1.2, presence_penalty=0.1, frequency_penalty=0.05, allowed=allowed)
    draw = dict(temperature=0.9, seeds=torch.tensor([1, 2, 3], device="cuda")) if sample else {}
    with torch.no_grad():
        dec = Mamba3LMDecoder(model, use_cuda_graph=graph, w4_group_size=w4, **FUSED)
        plain = Mamba3LMDecoder(model, w4_group_size=w4, **FUSED)
        if graph:
            dec.warmup_cuda_graph(dec.init_state(3, device="cuda"), n_warmup=1)
        for _ in range(2):  # again: a captured decoder starts over
            toks, lps, lengths = dec.generate(ids, new, prompt_lengths=torch.tensor([4, 1, 7]), **kw,
                                               **draw)
        assert toks.shape == lps.shape == (3, L + new)
        for b, p in enumerate(prompts):
            def args(n, b=b):
                return dict(kw, **(dict(temperature=0.9, seeds=draw["seeds"][b:b + 1],
                                        positions=torch.tensor([n], device="cuda")) if sample else {}))
            want, want_lp = by_hand(plain, p, new, kw=args)
            n = len(p) + new
            assert int(lengths[b]) == n and toks[b, :n].tolist() == want
            assert not toks[b, n:].any() and not lps[b, n:].any() and not lps[b, :len(p)].any()
            torch.testing.assert_close(lps[b, len(p):n].cpu(), torch.tensor(want_lp), rtol=1e-4, atol=1e-4)


def test_generate_stops_at_the_end_token():
    model = lm(seed=4)
    ids = torch.randint(0, 203, (4, 3), device="cuda")
    dec = Mamba3LMDecoder(model, **FUSED)
    free, _, _ = dec.generate(ids, 8)
    eos = int(free[0, 5])
    toks, lps, lengths = dec.generate(ids, 8, eos_token_id=eos)
    for b in range(4):
        gen = free[b, 3:].tolist()
        n = gen.index(eos) + 1 if eos in gen else 8
        assert int(lengths[b]) == 3 + n and toks[b, 3:3 + n].tolist() == gen[:n]
        assert not toks[b, 3 + n:].any() and not lps[b, 3 + n:].any()


def test_generate_keeps_to_the_vocabulary():
    """The head is padded to a multiple of 8: its last rows are no tokens."""
    model = lm(vocab=201)
    assert model.vocab_size == 208
    with torch.no_grad():
        model.lm_head.weight[201:] = model.lm_head.weight[:201].abs().max() * 100 * model.lm_head.weight[0].sign()
    toks, _, _ = Mamba3LMDecoder(model, **FUSED).generate(torch.zeros(5, 2, dtype=torch.long, device="cuda"), 10)
    assert int(toks.max()) < 201


def test_generate_edges_and_refusals():
    model = lm()
    dec = Mamba3LMDecoder(model, **FUSED)
    ids = torch.randint(0, 203, (2, 3), device="cuda")
    toks, lps, lengths = dec.generate(ids, 0)
    assert torch.equal(toks, ids) and lengths.tolist() == [3, 3] and not lps.any()
    toks, _, _ = dec.generate(torch.empty(0, 3, dtype=torch.long, device="cuda"), 4)
    assert toks.shape == (0, 7)
    for bad in (torch.full((2, 3), 203, device="cuda"), torch.full((2, 3), -1, device="cuda")):
        with pytest.raises(ValueError):
            dec.generate(bad, 2)
    for pl in ([0, 3], [1, 4]):
        with pytest.raises(ValueError):
            dec.generate(ids, 2, prompt_lengths=torch.tensor(pl))
    with pytest.raises(ValueError):
        dec.generate(ids, 2, eos_token_id=203)
    with pytest.raises(AssertionError):
        dec.generate(ids.cpu(), 2)
    with pytest.raises(ValueError):
        Mamba3Decoder(model.layers[0].mixer, w4_group_size=48, **FUSED)
    with pytest.raises(ValueError):
        Mamba3Decoder(model.layers[0].mixer, w4_group_size=64)
